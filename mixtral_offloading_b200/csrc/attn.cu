// Attention of new tokens over pages (hqm_paged_attention) and over whole packed prompts (hqm_prompt_attention): checks, tensor
// maps, and which kernel runs.
#include <math.h>

#include "attn.cuh"
#include "overlap.h"

namespace hqm {
namespace attn {
namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int sm_count() {
    static int counts[MAX_DEVICES];
    int& n = counts[current_device_slot()];
    if (n == 0) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) cudaGetLastError();
    }
    return n;
}

// Strides in elements.  Boxes start at 64 columns, 128-byte swizzle.
bool encode(CUtensorMap* to, const void* at, int rank, const cuuint64_t* dims, const int64_t* strides, const cuuint32_t* box, bool f16) {
    const EncodeTiledFn enc = (EncodeTiledFn)tma_encode_entry();
    if (!enc) return false;
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    cuuint64_t bytes[4];
    for (int i = 0; i < rank - 1; ++i) bytes[i] = (cuuint64_t)strides[i] * 2;
    return enc(to, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(at), dims, bytes, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Keys or values: `rows` positions of one head of one page (packed: of the one page that all of them are).  `across`: 64 columns
// after another in one box; else one box brings 64 columns.
bool encode_kv(CUtensorMap* to, const void* at, int D, int rows, cuuint64_t positions, cuuint64_t heads, cuuint64_t pages, int64_t position, int64_t head,
               int64_t page, bool across, bool f16) {
    if (across) {
        const cuuint64_t dims[5] = {64, positions, (cuuint64_t)D / 64, heads, pages};
        const int64_t strides[4] = {position, 64, head, page};
        const cuuint32_t box[5] = {64, (cuuint32_t)rows, (cuuint32_t)D / 64, 1, 1};
        return encode(to, at, 5, dims, strides, box, f16);
    }
    const cuuint64_t dims[4] = {(cuuint64_t)D, positions, heads, pages};
    const int64_t strides[3] = {position, head, page};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
    return encode(to, at, 4, dims, strides, box, f16);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check(const hqm_attention* c, bool paged, const char* what) {
    HQM_CHECK_ARG(c, "%s: null pointer", what);
    HQM_CHECK_ARG(c->tokens >= 0 && c->tokens <= INT32_MAX && c->sequences >= 0 && c->max_new >= 0, "%s: %lld tokens of %d sequences, at most %d each",
                  what, (long long)c->tokens, c->sequences, c->max_new);
    HQM_CHECK_ARG((c->head_dim == 64 || c->head_dim == 128) && (c->dtype == 0 || c->dtype == 1), "%s: head_dim %d (64 or 128), dtype %d (0 bf16, 1 fp16)",
                  what, c->head_dim, c->dtype);
    HQM_CHECK_ARG(c->n_kv_heads > 0 && c->n_heads > 0 && c->n_heads % c->n_kv_heads == 0 && c->n_heads / c->n_kv_heads <= MAX_GROUP,
                  "%s: %d query heads on %d key/value heads (a multiple, at most %d times)", what, c->n_heads, c->n_kv_heads, MAX_GROUP);
    HQM_CHECK_ARG(c->scale > 0.f && isfinite(c->scale), "%s: scale %g (positive)", what, (double)c->scale);
    if (paged) {
        const int64_t page_elements = (int64_t)c->n_kv_heads * c->page_size * c->head_dim;
        HQM_CHECK_ARG(c->page_size >= 16 && (c->page_size & (c->page_size - 1)) == 0 && c->pages > 0 && c->max_pages > 0 &&
                          c->table_stride >= c->max_pages && (int64_t)c->pages * c->page_size <= INT32_MAX && c->k_page >= page_elements &&
                          c->v_page >= page_elements,
                      "%s: %d pages of %d positions (a power of two, 16 or more), %lld and %lld elements apart, rows of %d pages", what, c->pages,
                      c->page_size, (long long)c->k_page, (long long)c->v_page, c->max_pages);
        HQM_CHECK_ARG((int64_t)c->max_pages * c->page_size <= INT32_MAX - TILE_KEYS, "%s: rows of %d pages of %d positions", what, c->max_pages, c->page_size);
    }
    if (c->tokens == 0 || c->sequences == 0 || c->max_new == 0) return HQM_OK;
    HQM_CHECK_ARG(c->out && c->q && c->k && c->v && c->cu_seqlens && (!paged || (c->block_table && c->kv_lens)), "%s: null pointer", what);
    const int64_t strides = c->q_token | c->q_head | (paged ? c->k_page | c->v_page : c->k_token | c->k_head | c->v_token | c->v_head);
    HQM_CHECK_ARG(strides % 8 == 0 && aligned16(c->q) && aligned16(c->k) && aligned16(c->v) && aligned16(c->out),
                  "%s: rows have to start on 16-byte boundaries", what);
    if (!paged) HQM_CHECK_ARG(c->k_token > 0 && c->k_head > 0 && c->v_token > 0 && c->v_head > 0, "%s: strides of keys and values have to be positive", what);
    const Stretch out = elements_at(c->out, c->tokens * c->n_heads * c->head_dim);
    const int64_t page_elements = (int64_t)c->n_kv_heads * c->page_size * c->head_dim;
    const bool shared = out.meets(rows_at(c->q, c->tokens, c->n_heads, c->q_token, c->q_head, c->head_dim)) ||
                        (paged ? Pages{c->k, c->pages, c->k_page, page_elements}.meets(out) || Pages{c->v, c->pages, c->v_page, page_elements}.meets(out)
                               : out.meets(rows_at(c->k, c->tokens, c->n_kv_heads, c->k_token, c->k_head, c->head_dim)) ||
                                     out.meets(rows_at(c->v, c->tokens, c->n_kv_heads, c->v_token, c->v_head, c->head_dim)));
    HQM_CHECK_ARG(!shared, "%s: out shares memory with what is read", what);
    return HQM_OK;
}

// Which kernels a call takes: attn_few.cu where its unit holds all new tokens of any sequence, else attn_tiles.cu.  Where the
// sequences beside the longest have few rows on average, both: those that fit a unit of attn_few.cu run there, at the
// rate of the memory, and do not fill a tile of 128 rows with four.  30 single tokens and 1, 2, 4, 8 chunks of up to 512, 32 on 8 heads of 128 (in
// front of every call the caches are overwritten): 85, 89, 103, 145 us by both, 93, 98, 116, 162 by attn_tiles.cu alone.  The rule asks for few
// rows beside ONE longest sequence, which is what the host knows: of those it takes the first two.
struct Kernels {
    bool few, tiles;
    static Kernels of(const hqm_attention* c, bool paged) {
        const int64_t group = c->n_heads / c->n_kv_heads, most = c->max_new < c->tokens ? c->max_new : c->tokens;
        if (most * group <= FEW_TILE) return {true, false};
        const bool mixed = paged && group <= FEW_TILE && (c->tokens - most) * group <= (int64_t)MIXED_ROWS * (c->sequences - 1);
        return {mixed && c->sequences > 1, true};
    }
};
// Whether units are cut.  Where there is a CTA for each and none is long, they are not: the blocks that a CTA then works through one
// after another cost less than the launch that joins pieces.  What is known here of the lengths are bounds: the table's rows,
// max_new (so a table whose rows are far wider than its sequences are long has its units cut); the units of a prompt have half as many
// blocks as the longest on average.  32 on 8 heads of 128, with pieces and
// whole: one token on 100 positions 8.6 and 6.6 us, on 300 8.7 and 8.3, on 500 9.0 and 10.5; 60 tokens behind 300 14.3 and 12.6, behind 500
// 15.2 and 16.3; a prompt of 250 tokens 14.9 and 11.7, of 500 17.4 and 15.0, of 700 20.8 and 18.2.
bool cuts(const hqm_attention* c, bool paged, int ctas, int per, int block, int most_blocks) {
    const int64_t most = c->max_new < c->tokens ? c->max_new : c->tokens;
    const int64_t positions = paged ? (int64_t)c->max_pages * c->page_size : most, blocks = (positions + block - 1) / block;
    const int64_t units = (c->tokens / per + c->sequences) * c->n_kv_heads;
    return blocks > 1 && (units > ctas || (paged ? blocks : (blocks + 1) / 2) > most_blocks);
}
size_t launch_bytes(int ctas, int rows, int D) { return record_bytes(ctas) + (piece_bytes(ctas, rows, D) + 255) / 256 * 256; }

int run(const hqm_attention* c, bool paged, const char* what, void* scratch, size_t scratch_bytes, void* stream) {
    if (int rc = check(c, paged, what)) return rc;
    if (c->tokens == 0 || c->sequences == 0 || c->max_new == 0) return HQM_OK;
    const int ctas = sm_count();
    HQM_CHECK_ARG(ctas > 0, "%s: no device", what);
    const size_t need = hqm_attention_scratch_bytes(c);
    if (!scratch || scratch_bytes < need) {
        set_error("%s: scratch too small (%zu < %zu)", what, scratch_bytes, need);
        return HQM_ERR_SCRATCH;
    }
    HQM_CHECK_ARG(aligned16(scratch), "%s: scratch has to be 16-byte aligned", what);
    const bool f16 = c->dtype == 1;
    const int D = c->head_dim;
    Args a{};
    a.q = (const uint16_t*)c->q;
    a.out = (uint16_t*)c->out;
    a.out_32 = (reinterpret_cast<uintptr_t>(c->out) & 31u) == 0;
    a.q_token = c->q_token;
    a.q_head = c->q_head;
    a.table = paged ? c->block_table : nullptr;
    a.table_stride = c->table_stride;
    a.cu = c->cu_seqlens;
    a.kv_lens = c->kv_lens;
    a.B = c->sequences;
    a.T = (int)c->tokens;
    a.n_kv = c->n_kv_heads;
    a.group = c->n_heads / c->n_kv_heads;
    a.n_pages = c->pages;
    a.max_pages = c->max_pages;
    if (paged)
        while ((1 << a.page_shift) < c->page_size) ++a.page_shift;
    a.scale_log2 = (float)((double)c->scale * 1.4426950408889634);
    Args few = a, tiles = a;
    uint8_t* at = (uint8_t*)scratch;
    auto place = [&](Args& to, int rows) {
        to.records = (int32_t*)at;
        to.pieces = (float*)(at + record_bytes(ctas));
        to.piece_rows = rows;
        at += launch_bytes(ctas, rows, D);
    };
    const Kernels k = Kernels::of(c, paged);
    few.cuts = cuts(c, paged, ctas, FEW_TILE / a.group > 0 ? FEW_TILE / a.group : 1, FEW_KEYS, FEW_WHOLE);
    tiles.cuts = cuts(c, paged, ctas, TILE_ROWS / 2 / a.group * 2, TILE_KEYS, TILES_WHOLE);
    few.rows_above = tiles.rows_above = 0;
    few.rows_upto = tiles.rows_upto = INT32_MAX;
    if (k.few && k.tiles) few.rows_upto = tiles.rows_above = FEW_TILE;
    // keys and values: rows of a box, and whether it brings all columns
    auto maps = [&](CUtensorMap* km, CUtensorMap* vm, int keys, bool across) {
        if (paged) {
            const int rows = c->page_size < keys ? c->page_size : keys;
            const int64_t head = (int64_t)c->page_size * D;
            return encode_kv(km, c->k, D, rows, c->page_size, c->n_kv_heads, c->pages, D, head, c->k_page, across, f16) &&
                   encode_kv(vm, c->v, D, rows, c->page_size, c->n_kv_heads, c->pages, D, head, c->v_page, across, f16);
        }
        return encode_kv(km, c->k, D, keys, c->tokens, c->n_kv_heads, 1, c->k_token, c->k_head, c->k_token * c->tokens, across, f16) &&
               encode_kv(vm, c->v, D, keys, c->tokens, c->n_kv_heads, 1, c->v_token, c->v_head, c->v_token * c->tokens, across, f16);
    };
    auto no_maps = [&]() {
        set_error("%s: the driver does not encode the tensor maps", what);
        return HQM_ERR_CUDA;
    };
    const cudaStream_t st = (cudaStream_t)stream;
    CUtensorMap qm, km, vm, kf, vf;
    if (k.tiles) {
        place(tiles, TILE_ROWS);
        // row = token * group + head: a box of all heads of a group and as many tokens as a tile holds
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.group, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->tokens};
        const int64_t strides[3] = {c->q_head, c->q_head * a.group, c->q_token};
        const cuuint32_t box[4] = {64, (cuuint32_t)a.group, 1, 128u / a.group};
        if (!maps(&km, &vm, TILE_KEYS, false) || !encode(&qm, c->q, 4, dims, strides, box, f16)) return no_maps();
    }
    if (k.few) {
        place(few, FEW_TILE);
        if (!maps(&kf, &vf, FEW_KEYS, true)) return no_maps();
    }
    const int rc = k.few && k.tiles ? launch_mixed(tiles, few, qm, km, vm, kf, vf, ctas, D, f16, st)
                   : k.few          ? launch_few(few, kf, vf, ctas, D, f16, st)
                                    : launch_tiles(tiles, qm, km, vm, ctas, D, f16, st);
    if (rc) return rc;
    if (!(k.tiles && tiles.cuts) && !(k.few && few.cuts)) return HQM_OK;
    return launch_join(k.tiles ? tiles : few, k.tiles && k.few ? &few : nullptr, ctas, D, f16, st);
}

}  // namespace
}  // namespace attn
}  // namespace hqm

extern "C" {

size_t hqm_attention_scratch_bytes(const hqm_attention* c) {
    using namespace hqm::attn;
    if (!c || c->n_kv_heads <= 0 || c->n_heads < c->n_kv_heads || (c->head_dim != 64 && c->head_dim != 128)) return 0;
    const int ctas = sm_count() > 0 ? sm_count() : 148;
    const Kernels k = Kernels::of(c, c->block_table != nullptr);
    return (k.tiles ? launch_bytes(ctas, TILE_ROWS, c->head_dim) : 0) + (k.few ? launch_bytes(ctas, FEW_TILE, c->head_dim) : 0);
}
int hqm_paged_attention(const hqm_attention* call, void* scratch, size_t scratch_bytes, void* stream) {
    return hqm::attn::run(call, true, "paged_attention", scratch, scratch_bytes, stream);
}
int hqm_prompt_attention(const hqm_attention* call, void* scratch, size_t scratch_bytes, void* stream) {
    return hqm::attn::run(call, false, "prompt_attention", scratch, scratch_bytes, stream);
}

}  // extern "C"
