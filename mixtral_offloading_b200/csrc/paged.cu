// A key/value cache in pages: block tables and slot maps from request lengths, and the append into pages.
//
// Tables.  The pages that nobody holds are a stack, free[0 .. count - 1].  Sequence b has len_b positions in the pages
// table[b][0 .. ceil(len_b / P) - 1].  n_b new tokens need ceil((len_b + n_b) / P) - ceil(len_b / P) pages more; with F_b the sum of
// what the sequences before b need, page i of them is free[count - 1 - (F_b + i)], and new token t of all has position
// len_b + t - cu_b and the slot (page of its position) * P + position % P.  All of it is two prefix sums over the sequences and a
// search per page and token.  Bound by latency: one CTA, which takes a token's page off the stack without waiting for the
// table; positions and slots of more than 4096 tokens are left to a second launch of as many CTAs as it takes (102000 tokens of 256
// sequences: 27 us in one launch of eight CTAs, 9 so).
//
// Append.  turn = position * theta^(-2 d / D) / 2 pi in 64 bits (a position of 10^5 leaves 32 bits with 10^-2 of an angle), its
// fraction in 32; (a, b) -> (a cos - b sin, b cos + a sin) in fp32, rounded once.  Bound by bytes: q in and out, k and v into
// their pages, sixteen at a time.
#include <math.h>

#include "common.cuh"
#include "kernels.cuh"
#include "overlap.h"
#include "shared_limit.h"

namespace hqm {
namespace {

constexpr int TABLE_THREADS = 512;
constexpr int64_t TABLE_ALONE = 4096;
constexpr int PAGES_AT_ONCE = 4;
constexpr int MAP_THREADS = 256, MAP_TOKENS = 4 * MAP_THREADS;
constexpr int MAX_SEQUENCES = 16384;         // three words of shared memory each

struct Tables {
    int32_t* table;
    int64_t stride;
    int32_t *lens, *free_pages, *free_count;
    const int32_t* change;                   // new lengths, or the lengths to keep
    int32_t *cu, *after, *positions, *slots, *status;
    int B, max_pages, page, capacity;        // capacity: of free_pages
    int64_t tokens;
    int maps;                                // positions and slots as well
};

__device__ __forceinline__ int64_t shift_up(int64_t v, int o) { return __shfl_up_sync(0xffffffffu, v, o); }

// Pages of `len` positions.  (In 32 bits, which ceil of 2^31 - 1 fits: a division of 64 bits takes some 600 cycles.)
__device__ __forceinline__ int pages_of(int len, int page) { return (int)(((uint32_t)len + page - 1) / (uint32_t)page); }

// The last i of 0 .. n - 1 with at[i] <= x (at is not decreasing, at[0] <= x): of equal ones the one whose range holds x.
__device__ __forceinline__ int range_of(const int32_t* at, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// TAKE: new tokens get their pages; else the pages behind `change` positions go back.
template <bool TAKE>
__global__ void __launch_bounds__(TABLE_THREADS) tables_kernel(const __grid_constant__ Tables p) {
    extern __shared__ int32_t words[];
    int32_t* s_cu = words;                   // B + 1: first new token
    int32_t* s_pg = words + p.B + 1;         // B + 1: first page that moves
    int32_t* s_len = words + 2 * (p.B + 1);
    __shared__ int64_t s_sum[2][TABLE_THREADS / 32];
    __shared__ int s_bad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) s_bad = 0;
    grid_launch_dependents();
    grid_dependency_wait();
    const int count = *p.free_count;
    __syncthreads();
    int64_t base[2] = {0, 0};                // tokens and pages of the sequences before this round's
    for (int b0 = 0; b0 < p.B; b0 += TABLE_THREADS) {
        const int b = b0 + threadIdx.x;
        int64_t v[2] = {0, 0};
        if (b < p.B) {
            const int len = p.lens[b], by = p.change[b];
            const int64_t to = TAKE ? (int64_t)len + by : by;
            const int64_t row = (int64_t)p.max_pages * p.page, most = row < INT32_MAX ? row : INT32_MAX;
            if (len < 0 || by < 0 || len > most || to > most || (!TAKE && by > len)) s_bad = 1;
            else {
                const int held = pages_of(len, p.page), then = pages_of((int)to, p.page);
                v[0] = TAKE ? by : 0;
                v[1] = TAKE ? then - held : held - then;
            }
            s_len[b] = len;
        }
        int64_t own[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            own[i] = v[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t up = shift_up(v[i], o);
                if (lane >= o) v[i] += up;
            }
            if (lane == 31) s_sum[i][warp] = v[i];
        }
        __syncthreads();
        int64_t all[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            int64_t before = base[i];
            for (int k = 0; k < TABLE_THREADS / 32; ++k) {
                if (k < warp) before += s_sum[i][k];
                all[i] += s_sum[i][k];
            }
            const int64_t at = before + v[i] - own[i];
            if (b < p.B) (i ? s_pg : s_cu)[b] = (int32_t)(at < INT32_MAX ? at : INT32_MAX);
            base[i] += all[i];
        }
        __syncthreads();
    }
    // all or nothing: 0; pages that are missing; -1: a length that no table row holds; -2: more tokens than the maps have rows
    int status = 0;
    if (s_bad) status = -1;
    else if (TAKE && base[0] > p.tokens) status = -2;
    else if (count < 0 || count > p.capacity || (!TAKE && base[1] > p.capacity - count)) status = -3;
    else if (TAKE && base[1] > count) status = (int)(base[1] - count < INT32_MAX ? base[1] - count : INT32_MAX);
    const int n_tokens = status == 0 ? (int)base[0] : 0, n_pages = status == 0 ? (int)base[1] : 0;
    const int tid = threadIdx.x;
    constexpr int all = TABLE_THREADS;
    __syncthreads();                         // the last read of lengths and count lies in front, their first write behind
    const int top = TAKE ? count - 1 : count + n_pages - 1;
    for (int i0 = tid; i0 < n_pages; i0 += PAGES_AT_ONCE * all) {
        int32_t *to[PAGES_AT_ONCE], moved[PAGES_AT_ONCE];
#pragma unroll
        for (int k = 0; k < PAGES_AT_ONCE; ++k) {
            const int i = i0 + k * all;
            if (i >= n_pages) continue;
            const int b = range_of(s_pg, p.B, i);
            int32_t* entry = p.table + (int64_t)b * p.stride + pages_of(TAKE ? s_len[b] : p.change[b], p.page) + (i - s_pg[b]);
            int32_t* place = p.free_pages + (top - i);
            to[k] = TAKE ? entry : place;
            moved[k] = TAKE ? *place : *entry;
        }
#pragma unroll
        for (int k = 0; k < PAGES_AT_ONCE; ++k)
            if (i0 + k * all < n_pages) *to[k] = moved[k];
    }
    if (TAKE) {
        for (int64_t t = tid; p.maps && t < p.tokens; t += all) {
            int position = -1, slot = -1;
            if (t < n_tokens) {
                const int b = range_of(s_cu, p.B, (int)t);
                const int len = s_len[b], held = pages_of(len, p.page);
                position = len + ((int)t - s_cu[b]);
                const int i = position / p.page;
                const int page = i < held ? p.table[(int64_t)b * p.stride + i] : p.free_pages[top - (s_pg[b] + i - held)];
                slot = (int)((int64_t)page * p.page + position % p.page);
            }
            p.positions[t] = position;
            p.slots[t] = slot;
        }
        for (int b = tid; b <= p.B; b += all) p.cu[b] = status != 0 ? 0 : (b < p.B ? s_cu[b] : n_tokens);
    }
    for (int b = tid; b < p.B; b += all) {
        const int then = status != 0 ? s_len[b] : (TAKE ? s_len[b] + p.change[b] : p.change[b]);
        if (TAKE) p.after[b] = then;
        p.lens[b] = then;
    }
    if (tid == 0) {
        if (status == 0) *p.free_count = TAKE ? count - n_pages : count + n_pages;
        *p.status = status;
    }
}

// Positions and slots from the offsets, lengths and table that tables_kernel leaves: MAP_TOKENS tokens per CTA.
__global__ void __launch_bounds__(MAP_THREADS) maps_kernel(const __grid_constant__ Tables p) {
    extern __shared__ int32_t words[];
    __shared__ int s_first, s_last;
    grid_launch_dependents();
    grid_dependency_wait();
    const int64_t t0 = (int64_t)blockIdx.x * MAP_TOKENS;
    const int n_tokens = p.cu[p.B];
    // the sequences of this CTA's tokens: their offsets in shared memory
    if (threadIdx.x < 2) {
        const int64_t t = threadIdx.x == 0 ? t0 : t0 + MAP_TOKENS - 1;
        const int at = range_of(p.cu, p.B, (int)(t < n_tokens - 1 ? t : (n_tokens > 0 ? n_tokens - 1 : 0)));
        (threadIdx.x == 0 ? s_first : s_last) = at;
    }
    __syncthreads();
    const int first = s_first, count = p.B > 0 ? s_last - first + 1 : 0;
    for (int i = threadIdx.x; i <= count; i += MAP_THREADS) words[i] = p.cu[first + i];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < MAP_TOKENS / MAP_THREADS; ++k) {
        const int64_t t = t0 + k * MAP_THREADS + threadIdx.x;
        if (t >= p.tokens) return;
        int position = -1, slot = -1;
        if (t < n_tokens) {
            const int i = range_of(words, count, (int)t), b = first + i;
            position = p.after[b] - (words[i + 1] - (int)t);
            slot = (int)((int64_t)p.table[(int64_t)b * p.stride + position / p.page] * p.page + position % p.page);
        }
        p.positions[t] = position;
        p.slots[t] = slot;
    }
}

int launch_tables(Tables p, bool take, cudaStream_t st) {
    static SharedLimits limits[3];
    const size_t bytes = (size_t)(3 * p.B + 2) * sizeof(int32_t), map_bytes = (size_t)(p.B + 1) * sizeof(int32_t);
    void (*kernel)(const Tables) = take ? tables_kernel<true> : tables_kernel<false>;
    p.maps = p.tokens <= TABLE_ALONE;
    if ((bytes > 40 * 1024 && !allow_shared(kernel, limits[take], bytes)) || (map_bytes > 40 * 1024 && !allow_shared(maps_kernel, limits[2], map_bytes))) {
        set_error("paged tables: %d sequences want %zu bytes of shared memory", p.B, bytes);
        return HQM_ERR_CUDA;
    }
    HQM_CUDA(launch_overlapped(kernel, 1, TABLE_THREADS, bytes, st, p));
    HQM_LAUNCH_CHECK();
    if (p.maps) return HQM_OK;
    HQM_CUDA(launch_overlapped(maps_kernel, (int)((p.tokens + MAP_TOKENS - 1) / MAP_TOKENS), MAP_THREADS, map_bytes, st, p));
    HQM_LAUNCH_CHECK();
    return HQM_OK;
}

// ---- append ---------------------------------------------------------------------------------------------------------
struct Append {
    uint16_t *q_out, *k_out;                 // (T, n_heads, D); (T, n_kv, D) or null
    const uint16_t *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    uint16_t *k_pages, *v_pages;             // (pages, n_kv, page, D)
    int64_t k_page, v_page;                  // strides of a page
    const int32_t *positions, *slots;
    int T, n_heads, n_kv, pages, page;
    double turns[64];                        // theta^(-2 d / D) / 2 pi
};
constexpr int APPEND_THREADS = 128, APPEND_AHEAD = 2;        // see rope_append_paged_kernel

template <bool F16>
__device__ __forceinline__ void rotate8(const uint4& lo, const uint4& hi, const float2* cs, uint4& out_lo, uint4& out_hi) {
    const uint32_t* a = &lo.x;
    const uint32_t* b = &hi.x;
    uint32_t* x = &out_lo.x;
    uint32_t* y = &out_hi.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float u[2], w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint16_t ab = (uint16_t)(a[i] >> (16 * e)), bb = (uint16_t)(b[i] >> (16 * e));
            const float av = F16 ? f16_bits_to_float(ab) : bf16_bits_to_float(ab), bv = F16 ? f16_bits_to_float(bb) : bf16_bits_to_float(bb);
            const float2 c = cs[2 * i + e];
            u[e] = av * c.x - bv * c.y;
            w[e] = bv * c.x + av * c.y;
        }
        if constexpr (F16) {
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x[i]) : "f"(u[1]), "f"(u[0]));
            asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y[i]) : "f"(w[1]), "f"(w[0]));
        } else {
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(x[i]) : "f"(u[1]), "f"(u[0]));
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y[i]) : "f"(w[1]), "f"(w[0]));
        }
    }
}

// One CTA per token.  The bytes on their way set the time: 9121 tokens, 32 and 8 heads of 128, 224 MB: 49.5 us with 256 threads and one
// item ahead, 41.3 with 128 threads and two at once (5.4 TB/s), 42.8 with three, 45.5 with 192 threads and two.
template <int D, bool F16>
__global__ void __launch_bounds__(APPEND_THREADS) rope_append_paged_kernel(const __grid_constant__ Append p, int* error_flag) {
    constexpr int HALF = D / 2, VEC = HALF / 8;
    __shared__ float2 cs[HALF];
    grid_launch_dependents();
    grid_dependency_wait();
    const int t = blockIdx.x;
    // items: pairs of eight columns of q, of k, then sixteen columns of v
    const int q_items = p.n_heads * VEC, k_items = p.n_kv * VEC, items = q_items + 2 * k_items;
    auto load = [&](int i, uint4& lo, uint4& hi) {
        if (i < q_items + k_items) {
            const bool is_q = i < q_items;
            const int j = is_q ? i : i - q_items, head = j / VEC, d = (j % VEC) * 8;
            const uint16_t* src = is_q ? p.q + t * p.q_token + head * p.q_head + d : p.k + t * p.k_token + head * p.k_head + d;
            lo = *reinterpret_cast<const uint4*>(src);
            hi = *reinterpret_cast<const uint4*>(src + HALF);
        } else {
            const int j = i - q_items - k_items, head = j / VEC, d = (j % VEC) * 16;
            const uint16_t* src = p.v + t * p.v_token + head * p.v_head + d;
            lo = *reinterpret_cast<const uint4*>(src);
            hi = *reinterpret_cast<const uint4*>(src + 8);
        }
    };
    // items of a thread are on their way together, the first ones while the slot comes and the angles are formed
    uint4 lo[APPEND_AHEAD], hi[APPEND_AHEAD];
    auto load_from = [&](int i0) {
#pragma unroll
        for (int k = 0; k < APPEND_AHEAD; ++k)
            if (i0 + k * APPEND_THREADS < items) load(i0 + k * APPEND_THREADS, lo[k], hi[k]);
    };
    const int slot = p.slots[t];
    const int position = p.positions[t];
    load_from(threadIdx.x);
    if (slot < 0) return;
    if (slot >= p.pages * (int64_t)p.page) {
        if (threadIdx.x == 0 && error_flag) atomicExch(error_flag, 2);
        return;
    }
    const int page = slot / p.page, row = slot % p.page;
    uint16_t* const k_row = p.k_pages + page * p.k_page + (int64_t)row * D;
    uint16_t* const v_row = p.v_pages + page * p.v_page + (int64_t)row * D;
    const int64_t head_stride = (int64_t)p.page * D;
    if (threadIdx.x < HALF) {
        double turn = (double)position * p.turns[threadIdx.x];
        turn -= rint(turn);
        float sn, c;
        sincospif((float)(2.0 * turn), &sn, &c);
        cs[threadIdx.x] = make_float2(c, sn);
    }
    __syncthreads();
    auto store = [&](int i, const uint4& lo, const uint4& hi) {
        if (i < q_items + k_items) {
            const bool is_q = i < q_items;
            const int j = is_q ? i : i - q_items, head = j / VEC, d = (j % VEC) * 8;
            uint16_t* dst = is_q ? p.q_out + ((int64_t)t * p.n_heads + head) * D + d : k_row + head * head_stride + d;
            uint4 a, b;
            rotate8<F16>(lo, hi, cs + d, a, b);
            *reinterpret_cast<uint4*>(dst) = a;
            *reinterpret_cast<uint4*>(dst + HALF) = b;
            if (!is_q && p.k_out) {
                dst = p.k_out + ((int64_t)t * p.n_kv + head) * D + d;
                *reinterpret_cast<uint4*>(dst) = a;
                *reinterpret_cast<uint4*>(dst + HALF) = b;
            }
        } else {
            const int j = i - q_items - k_items, head = j / VEC, d = (j % VEC) * 16;
            *reinterpret_cast<uint4*>(v_row + head * head_stride + d) = lo;
            *reinterpret_cast<uint4*>(v_row + head * head_stride + d + 8) = hi;
        }
    };
    for (int i0 = threadIdx.x; i0 < items; i0 += APPEND_AHEAD * APPEND_THREADS) {
        if (i0 != threadIdx.x) load_from(i0);
#pragma unroll
        for (int k = 0; k < APPEND_AHEAD; ++k)
            if (i0 + k * APPEND_THREADS < items) store(i0 + k * APPEND_THREADS, lo[k], hi[k]);
    }
}

bool power_of_two(int v) { return v > 0 && (v & (v - 1)) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_tables(const char* what, const void* table, int64_t stride, const void* lens, const void* free_pages, const void* free_count,
                 const void* change, const void* status, int32_t sequences, int32_t max_pages, int32_t page_size, int32_t capacity) {
    HQM_CHECK_ARG(sequences >= 0 && sequences <= MAX_SEQUENCES, "%s: %d sequences (at most %d)", what, sequences, MAX_SEQUENCES);
    HQM_CHECK_ARG(max_pages > 0 && stride >= max_pages && page_size > 0 && capacity > 0 && (int64_t)capacity * page_size <= INT32_MAX,
                  "%s: %d pages of %d positions, rows of %d pages (stride %lld)", what, capacity, page_size, max_pages, (long long)stride);
    HQM_CHECK_ARG(free_pages && free_count && status && (sequences == 0 || (table && lens && change)), "%s: null pointer", what);
    return HQM_OK;
}

}  // namespace
}  // namespace hqm

extern "C" {

int hqm_paged_reserve(int32_t* block_table, int64_t table_stride, int32_t* kv_lens, const int32_t* free_pages, int32_t* free_count,
                      const int32_t* new_lens, int32_t* cu_seqlens, int32_t* kv_lens_after, int32_t* positions, int32_t* slots,
                      int32_t* status, int32_t sequences, int32_t max_pages, int32_t page_size, int32_t capacity, int64_t tokens,
                      void* stream) {
    using namespace hqm;
    if (int rc = check_tables("paged_reserve", block_table, table_stride, kv_lens, free_pages, free_count, new_lens, status, sequences, max_pages,
                              page_size, capacity))
        return rc;
    HQM_CHECK_ARG(tokens >= 0 && tokens <= INT32_MAX, "paged_reserve: %lld tokens", (long long)tokens);
    HQM_CHECK_ARG(cu_seqlens && (sequences == 0 || kv_lens_after) && (tokens == 0 || (positions && slots)), "paged_reserve: null pointer");
    const Tables p{block_table, table_stride, kv_lens, const_cast<int32_t*>(free_pages), free_count, new_lens, cu_seqlens, kv_lens_after,
                   positions, slots, status, sequences, max_pages, page_size, capacity, tokens, 0};
    return launch_tables(p, true, (cudaStream_t)stream);
}

int hqm_paged_truncate(const int32_t* block_table, int64_t table_stride, int32_t* kv_lens, int32_t* free_pages, int32_t* free_count,
                       const int32_t* keep, int32_t* status, int32_t sequences, int32_t max_pages, int32_t page_size, int32_t capacity,
                       void* stream) {
    using namespace hqm;
    if (int rc = check_tables("paged_truncate", block_table, table_stride, kv_lens, free_pages, free_count, keep, status, sequences, max_pages,
                              page_size, capacity))
        return rc;
    const Tables p{const_cast<int32_t*>(block_table), table_stride, kv_lens, free_pages, free_count, keep, nullptr, nullptr, nullptr, nullptr,
                   status, sequences, max_pages, page_size, capacity, 0, 0};
    return launch_tables(p, false, (cudaStream_t)stream);
}

int hqm_rope_append_paged(const hqm_paged_append* a, void* stream) {
    using namespace hqm;
    HQM_CHECK_ARG(a, "rope_append_paged: null pointer");
    HQM_CHECK_ARG(a->tokens >= 0 && a->tokens <= INT32_MAX, "rope_append_paged: %lld tokens", (long long)a->tokens);
    HQM_CHECK_ARG((a->head_dim == 64 || a->head_dim == 128) && (a->dtype == 0 || a->dtype == 1) && a->n_heads > 0 && a->n_kv_heads > 0,
                  "rope_append_paged: head_dim %d (64 or 128), dtype %d (0 bf16, 1 fp16), %d / %d heads", a->head_dim, a->dtype, a->n_heads,
                  a->n_kv_heads);
    const int64_t page_elements = (int64_t)a->n_kv_heads * a->page_size * a->head_dim;
    HQM_CHECK_ARG(a->pages > 0 && power_of_two(a->page_size) && (int64_t)a->pages * a->page_size <= INT32_MAX && a->k_page >= page_elements &&
                      a->v_page >= page_elements,
                  "rope_append_paged: %d pages of %d positions (a power of two), %lld and %lld elements apart", a->pages, a->page_size,
                  (long long)a->k_page, (long long)a->v_page);
    const double theta = (double)a->rope_theta + (double)a->rope_theta_low;      // (2^-25 of theta turns a position of 10^6 by 10^-3)
    HQM_CHECK_ARG(theta > 0.0 && isfinite(theta), "rope_append_paged: theta %g", theta);
    if (a->tokens == 0) return HQM_OK;
    HQM_CHECK_ARG(a->q_out && a->q && a->k && a->v && a->k_pages && a->v_pages && a->positions && a->slots, "rope_append_paged: null pointer");
    const int64_t strides = a->q_token | a->q_head | a->k_token | a->k_head | a->v_token | a->v_head | a->k_page | a->v_page;
    HQM_CHECK_ARG(strides % 8 == 0 && aligned16(a->q_out) && aligned16(a->k_out) && aligned16(a->q) && aligned16(a->k) && aligned16(a->v) && aligned16(a->k_pages) &&
                      aligned16(a->v_pages),
                  "rope_append_paged: rows have to start on 16-byte boundaries");
    // in place is safe, a thread reads what it is about to write; any other meeting is between threads
    const Stretch q = rows_at(a->q, a->tokens, a->n_heads, a->q_token, a->q_head, a->head_dim), q_out = elements_at(a->q_out, a->tokens * a->n_heads * a->head_dim);
    const Stretch k = rows_at(a->k, a->tokens, a->n_kv_heads, a->k_token, a->k_head, a->head_dim), v = rows_at(a->v, a->tokens, a->n_kv_heads, a->v_token, a->v_head, a->head_dim);
    const Stretch k_out = elements_at(a->k_out, a->k_out ? a->tokens * a->n_kv_heads * a->head_dim : 0);
    const bool q_in_place = a->q_out == a->q && (a->tokens == 1 || a->q_token == (int64_t)a->n_heads * a->head_dim) && (a->n_heads == 1 || a->q_head == a->head_dim);
    const bool k_in_place = a->k_out == a->k && (a->tokens == 1 || a->k_token == (int64_t)a->n_kv_heads * a->head_dim) && (a->n_kv_heads == 1 || a->k_head == a->head_dim);
    HQM_CHECK_ARG((q_in_place || !q_out.meets(q)) && !q_out.meets(k) && !q_out.meets(v), "rope_append_paged: the rotated q shares memory with what is read");
    HQM_CHECK_ARG(!a->k_out || ((k_in_place || !k_out.meets(k)) && !k_out.meets(q) && !k_out.meets(v) && !k_out.meets(q_out)),
                  "rope_append_paged: the rotated k shares memory with what is read, or with the rotated q");
    const Pages pools[2] = {{a->k_pages, a->pages, a->k_page, page_elements}, {a->v_pages, a->pages, a->v_page, page_elements}};
    HQM_CHECK_ARG(!pools[0].meets(pools[1]), "rope_append_paged: a page of keys shares memory with one of values");
    for (const Pages& pool : pools)
        HQM_CHECK_ARG(!pool.meets(q) && !pool.meets(k) && !pool.meets(v) && !pool.meets(q_out) && !pool.meets(k_out),
                      "rope_append_paged: a page shares memory with what is rotated");
    Append p{(uint16_t*)a->q_out, (uint16_t*)a->k_out, (const uint16_t*)a->q, (const uint16_t*)a->k, (const uint16_t*)a->v, a->q_token, a->q_head, a->k_token,
             a->k_head, a->v_token, a->v_head, (uint16_t*)a->k_pages, (uint16_t*)a->v_pages, a->k_page, a->v_page, a->positions, a->slots,
             (int)a->tokens, a->n_heads, a->n_kv_heads, a->pages, a->page_size, {}};
    const double step = pow(theta, -2.0 / a->head_dim);
    double f = 1.0 / (2.0 * 3.14159265358979323846);
    for (int d = 0; d < a->head_dim / 2; ++d, f *= step) p.turns[d] = f;
    const int grid = (int)a->tokens;
    const cudaStream_t st = (cudaStream_t)stream;
    if (a->head_dim == 128)
        HQM_CUDA(launch_overlapped(a->dtype ? rope_append_paged_kernel<128, true> : rope_append_paged_kernel<128, false>, grid, APPEND_THREADS, 0,
                                   st, p, tc_error_ptr()));
    else
        HQM_CUDA(launch_overlapped(a->dtype ? rope_append_paged_kernel<64, true> : rope_append_paged_kernel<64, false>, grid, APPEND_THREADS, 0,
                                   st, p, tc_error_ptr()));
    HQM_LAUNCH_CHECK();
    return HQM_OK;
}

}  // extern "C"
