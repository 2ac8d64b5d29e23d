// Attention of new tokens over pages (hqm_paged_attention) and over whole packed prompts (hqm_prompt_attention): checks, tensor
// maps, and which kernel runs.
#include <math.h>

#include "attn.cuh"

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

// Boxes of 64 x y x z x w elements, 128-byte swizzle; strides in elements.
bool encode(CUtensorMap* to, const void* at, const cuuint64_t (&dims)[4], const int64_t (&strides)[3], int y, int z, int w, bool f16) {
    const EncodeTiledFn enc = (EncodeTiledFn)tma_encode_entry();
    if (!enc) return false;
    const cuuint32_t ones[4] = {1, 1, 1, 1}, box[4] = {64, (cuuint32_t)y, (cuuint32_t)z, (cuuint32_t)w};
    const cuuint64_t bytes[3] = {(cuuint64_t)strides[0] * 2, (cuuint64_t)strides[1] * 2, (cuuint64_t)strides[2] * 2};
    return enc(to, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(at), dims, bytes, box, ones,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
        HQM_CHECK_ARG((int64_t)c->max_pages * c->page_size <= INT32_MAX, "%s: rows of %d pages of %d positions", what, c->max_pages, c->page_size);
    }
    if (c->tokens == 0 || c->sequences == 0 || c->max_new == 0) return HQM_OK;
    HQM_CHECK_ARG(c->out && c->q && c->k && c->v && c->cu_seqlens && (!paged || (c->block_table && c->kv_lens)), "%s: null pointer", what);
    const int64_t strides = c->q_token | c->q_head | (paged ? c->k_page | c->v_page : c->k_token | c->k_head | c->v_token | c->v_head);
    HQM_CHECK_ARG(strides % 8 == 0 && aligned16(c->q) && aligned16(c->k) && aligned16(c->v) && aligned16(c->out),
                  "%s: rows have to start on 16-byte boundaries", what);
    if (!paged) HQM_CHECK_ARG(c->k_token > 0 && c->k_head > 0 && c->v_token > 0 && c->v_head > 0, "%s: strides of keys and values have to be positive", what);
    return HQM_OK;
}

// Whether a unit of attn_few.cu holds all new tokens of any sequence.
bool few_rows(const hqm_attention* c) { return (int64_t)c->max_new * (c->n_heads / c->n_kv_heads) <= FEW_TILE; }
int rows_of_piece(const hqm_attention* c) { return few_rows(c) ? FEW_TILE : TILE_ROWS; }

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
    a.records = (int32_t*)scratch;
    a.pieces = (float*)((uint8_t*)scratch + record_bytes(ctas));
    a.piece_rows = rows_of_piece(c);
    CUtensorMap qm, km, vm;
    const bool few = few_rows(c);
    const int keys = few ? FEW_KEYS : TILE_KEYS, box = paged && c->page_size < keys ? c->page_size : keys;
    bool ok;
    if (paged) {
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)c->page_size, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->pages};
        const int64_t head = (int64_t)c->page_size * D;
        ok = encode(&km, c->k, dims, {(int64_t)D, head, c->k_page}, box, 1, 1, f16) && encode(&vm, c->v, dims, {(int64_t)D, head, c->v_page}, box, 1, 1, f16);
    } else {
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)c->tokens, (cuuint64_t)c->n_kv_heads, 1};
        ok = encode(&km, c->k, dims, {c->k_token, c->k_head, c->k_token * c->tokens}, box, 1, 1, f16) && encode(&vm, c->v, dims, {c->v_token, c->v_head, c->v_token * c->tokens}, box, 1, 1, f16);
    }
    if (ok && !few) {
        // row = token * group + head: a box of all heads of a group and as many tokens as a tile holds
        const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)a.group, (cuuint64_t)c->n_kv_heads, (cuuint64_t)c->tokens};
        ok = encode(&qm, c->q, dims, {c->q_head, c->q_head * a.group, c->q_token}, a.group, 1, 128 / a.group, f16);
    }
    if (!ok) {
        set_error("%s: the driver does not encode the tensor maps", what);
        return HQM_ERR_CUDA;
    }
    const cudaStream_t st = (cudaStream_t)stream;
    if (int rc = few ? launch_few(a, km, vm, ctas, D, f16, st) : launch_tiles(a, qm, km, vm, ctas, D, f16, st)) return rc;
    return launch_join(a, ctas, D, f16, st);
}

}  // namespace
}  // namespace attn
}  // namespace hqm

extern "C" {

size_t hqm_attention_scratch_bytes(const hqm_attention* c) {
    using namespace hqm::attn;
    if (!c) return 0;
    const int ctas = sm_count() > 0 ? sm_count() : 148;
    return record_bytes(ctas) + piece_bytes(ctas, rows_of_piece(c), c->head_dim);
}
int hqm_paged_attention(const hqm_attention* call, void* scratch, size_t scratch_bytes, void* stream) {
    return hqm::attn::run(call, true, "paged_attention", scratch, scratch_bytes, stream);
}
int hqm_prompt_attention(const hqm_attention* call, void* scratch, size_t scratch_bytes, void* stream) {
    return hqm::attn::run(call, false, "prompt_attention", scratch, scratch_bytes, stream);
}

}  // extern "C"
