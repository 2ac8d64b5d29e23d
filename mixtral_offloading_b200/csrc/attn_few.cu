// Attention of a few rows per key/value head (single tokens, short continuations) over pages of keys and values, and the pass
// that joins pieces of cut units for every attention kernel of the library.
//
//     out = softmax(q k^T scale) v,   2^(x log2 e) for exp, running maximum and total per row
//
// Bound by the bytes of keys and values: 4 D per position and key/value head.  One CTA per SM; a warp keeps a ring of stages
// full with tiled copies (64 positions of K and V each), eight warps work on them, two stages at a time, sixteen positions per
// warp.  Each warp has its own running maximum, total and sums, so that nothing is exchanged before the end of a unit.  The
// products go through mma.sync m16n8k16: with 16 rows at the most the matrix unit of tcgen05 would work on 128 rows of which
// seven eighths are padding, and the bytes, not the products, set the time.
#include <type_traits>

#include "attn.cuh"
#include "shared_limit.h"
#include "tc_common.cuh"

namespace hqm {
namespace attn {
namespace {

constexpr int CONSUMERS = 8;
constexpr int THREADS = 32 * (CONSUMERS + 1);
constexpr int STAGES = 4;
static_assert(STAGES % 2 == 0, "the halves of the warps take turns: a buffer belongs to one half, or that one would skip every other phase");
constexpr int UNIT_EXTRA = 1;          // what a unit costs beside its blocks, in blocks

template <int D>
struct Shared {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = FEW_KEYS * 128 * HALVES;          // 64 positions: boxes of [64 columns][rows of a box][128 bytes], 128-byte swizzle
    alignas(1024) unsigned char ring[STAGES][2][TILE];            // K, V
    float sums[CONSUMERS][FEW_TILE][D];
    float top[CONSUMERS][FEW_TILE], total[CONSUMERS][FEW_TILE];
    uint64_t full[STAGES], empty[STAGES];
    Run run;
};

// All columns of `rows` positions: [64 columns][rows][128 bytes].
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int row, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(0), "r"(row), "r"(head), "r"(page), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void sync_consumers() { asm volatile("bar.sync 1, %0;" ::"n"(32 * CONSUMERS) : "memory"); }

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1) attn_few_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                                                              const __grid_constant__ Args a, int* error_flag) {
    extern __shared__ __align__(1024) unsigned char raw[];
    using S = Shared<D>;
    S& sh = *reinterpret_cast<S*>(raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Cut how(FEW_TILE / a.group, FEW_KEYS_LOG, UNIT_EXTRA);
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            tc::mbar_init(&sh.full[i], 1);
            tc::mbar_init(&sh.empty[i], CONSUMERS / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&km);
        prefetch_map(&vm);
    }
    grid_launch_dependents();
    grid_dependency_wait();
    if (warp == 0) {
        const Run r = find_run(a, how, blockIdx.x, gridDim.x);
        if (lane == 0) sh.run = r;
    }
    __syncthreads();
    const Run run = sh.run;
    Walk w(a, run, how);
    bool ok = true;
    const int rows = a.table ? min(1 << a.page_shift, FEW_KEYS) : FEW_KEYS, boxes = FEW_KEYS / rows;       // of a box, per block
    if (warp == CONSUMERS) {
        // ---- the copies: lane i brings box i of a stage, K and V ----
        uint32_t at = 0;
        while (w.next() && ok) {
            const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
            // of block j; read one block ahead of the copies
            auto place = [&](int j, int& row, int& page) {
                const int key = j * FEW_KEYS + lane * rows;
                row = w.s.q0 + key;
                page = 0;
                if (!a.table || lane >= boxes || key >= w.s.kv) return;
                page = min((uint32_t)table[key >> a.page_shift], (uint32_t)a.n_pages);           // outside the pool: zeros
                row = key & ((1 << a.page_shift) - 1);
            };
            int row, page, next_row = 0, next_page = 0;
            place(w.j0, row, page);
            for (int j = w.j0; j < w.j1 && ok; ++j, ++at, row = next_row, page = next_page) {
                if (j + 1 < w.j1) place(j + 1, next_row, next_page);
                const int stage = at % STAGES;
                if (at >= STAGES) ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh.empty[stage], (at / STAGES - 1) & 1));
                if (!ok) break;
                const int live = min(boxes, (max(w.s.kv - j * FEW_KEYS, 0) + rows - 1) / rows);  // boxes that hold positions of the sequence
                const uint32_t bar = tc::smem_u32(&sh.full[stage]);
                if (lane == 0) expect(bar, (uint32_t)live * rows * 128 * S::HALVES * 2);
                __syncwarp();
                if (lane < live) {
                    copy_box(tc::smem_u32(sh.ring[stage][0] + lane * rows * 128 * S::HALVES), &km, row, w.h, page, bar);
                    copy_box(tc::smem_u32(sh.ring[stage][1] + lane * rows * 128 * S::HALVES), &vm, row, w.h, page, bar);
                }
                __syncwarp();
            }
        }
        // no copy may be on its way when the CTA ends
        for (uint32_t k = at < STAGES ? 0 : at - STAGES; k < at; ++k) tc::mbar_wait(&sh.full[k % STAGES], (k / STAGES) & 1);
        if (!ok && lane == 0 && error_flag) atomicExch(error_flag, 1);
        return;
    }
    // ---- the products ----
    const int half = warp >> 2, strip = (warp & 3) * 16;                   // stages of this half, positions within a stage
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;                         // rows r0 and r0 + 8, columns c0, c0 + 1 of an 8-wide tile
    // where position `key` of a stage lies, its first 64 columns; the next 64 are `across` bytes further on
    auto key_at = [&](int key) { return (uint32_t)(((key & ~(rows - 1)) * S::HALVES + (key & (rows - 1))) * 128); };
    const int across = rows * 128;
    const int krow = strip + (lane & 7) + ((lane >> 4) << 3), kch = (lane >> 3) & 1, vrow = strip + (lane & 15), vch = lane >> 4;
    const uint32_t k_off = key_at(krow), v_off = key_at(vrow);
    uint32_t at = 0;
    bool cut = false;
    while (w.next()) {
        const int tok0 = w.first_token(), n_rows = w.tokens() * a.group;
        uint32_t qf[D / 16][4];
        int limit[2];                                                      // positions that the two rows see
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + 8 * i, tok = tok0 + r / a.group;
            limit[i] = r < n_rows ? w.s.before + tok + 1 : 0;
            const uint16_t* src = a.q + (int64_t)(w.s.q0 + tok) * a.q_token + (int64_t)(w.h * a.group + r % a.group) * a.q_head + c0;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][i] = r < n_rows ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
                qf[k][i + 2] = r < n_rows ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f};
        for (int j = w.j0; j < w.j1; ++j, ++at) {
            if ((int)(at & 1) != half) continue;
            const int stage = at % STAGES;
            ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&sh.full[stage], (at / STAGES) & 1));
            const uint32_t kt = tc::smem_u32(sh.ring[stage][0]) + k_off, vt = tc::smem_u32(sh.ring[stage][1]) + v_off;
            const int key0 = j * FEW_KEYS + strip;
            if (key0 < w.s.kv) {
                float s[2][4] = {};
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t b[4];
                    const int ch = (2 * k + kch) & 7;
                    ldsm(b, kt + (k >> 2) * across + ((ch ^ (krow & 7)) << 4));
                    mma<F16>(s[0], qf[k], b[0], b[1]);
                    mma<F16>(s[1], qf[k], b[2], b[3]);
                }
                float now[2] = {top[0], top[1]};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 8 * t + c0 + (e & 1);
                        s[t][e] = key < limit[e >> 1] ? s[t][e] * a.scale_log2 : -INFINITY;
                        now[e >> 1] = fmaxf(now[e >> 1], s[t][e]);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 1));
                    now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 2));
                }
                if (__any_sync(0xffffffffu, now[0] != top[0] || now[1] != top[1])) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float f = now[i] == top[i] ? 1.f : ex2(top[i] - now[i]);      // (no -inf less -inf)
                        total[i] *= f;
#pragma unroll
                        for (int d = 0; d < D / 8; ++d) {
                            o[d][2 * i] *= f;
                            o[d][2 * i + 1] *= f;
                        }
                        top[i] = now[i];
                    }
                }
                const float base[2] = {top[0] == -INFINITY ? 0.f : top[0], top[1] == -INFINITY ? 0.f : top[1]};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][e] = ex2(s[t][e] - base[e >> 1]);
                        total[e >> 1] += s[t][e];
                    }
                const uint32_t p[4] = {pack2(s[0][0], s[0][1], F16), pack2(s[0][2], s[0][3], F16), pack2(s[1][0], s[1][1], F16),
                                       pack2(s[1][2], s[1][3], F16)};
                // what lies behind the sequence is anything, also NaN, which no weight of zero takes away
                const int past = key0 + 16 - w.s.kv;
                const int k0 = key0 + c0;
                const uint32_t m0 = past <= 0 ? 0xffffffffu : (k0 < w.s.kv ? 0xffffu : 0u) | (k0 + 1 < w.s.kv ? 0xffff0000u : 0u);
                const uint32_t m1 = past <= 0 ? 0xffffffffu : (k0 + 8 < w.s.kv ? 0xffffu : 0u) | (k0 + 9 < w.s.kv ? 0xffff0000u : 0u);
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    uint32_t b[4];
                    const int ch = (2 * d + vch) & 7;
                    ldsm_t(b, vt + (d >> 2) * across + ((ch ^ (vrow & 7)) << 4));
                    mma<F16>(o[2 * d], p, b[0] & m0, b[1] & m1);
                    mma<F16>(o[2 * d + 1], p, b[2] & m0, b[3] & m1);
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh.empty[stage]);
        }
        // ---- the eight warps' sums of this part become one ----
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            total[i] += __shfl_xor_sync(0xffffffffu, total[i], 1);
            total[i] += __shfl_xor_sync(0xffffffffu, total[i], 2);
        }
        sync_consumers();                                                  // the part before has been read
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if ((lane & 3) == 0) {
                sh.top[warp][r0 + 8 * i] = top[i];
                sh.total[warp][r0 + 8 * i] = total[i];
            }
            if (r0 + 8 * i < n_rows)
#pragma unroll
                for (int d = 0; d < D / 8; ++d)
                    *reinterpret_cast<float2*>(&sh.sums[warp][r0 + 8 * i][8 * d + c0]) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
        }
        sync_consumers();
        const bool whole = w.whole();
        float* piece = whole ? nullptr : piece_at<D>(a, blockIdx.x, w.j0 == 0);
        for (int i = threadIdx.x; i < n_rows * (D / 2); i += 32 * CONSUMERS) {
            const int r = i / (D / 2), d = (i % (D / 2)) * 2;
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < CONSUMERS; ++k) m = fmaxf(m, sh.top[k][r]);
            float l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int k = 0; k < CONSUMERS; ++k) {
                const float t = sh.top[k][r], f = t == -INFINITY ? 0.f : ex2(t - m);
                const float2 v = *reinterpret_cast<const float2*>(&sh.sums[k][r][d]);
                l += f * sh.total[k][r];
                x += f * v.x;
                y += f * v.y;
            }
            if (whole) {
                const float inv = m == -INFINITY ? 0.f : 1.f / l;
                const int64_t row = (int64_t)(w.s.q0 + tok0 + r / a.group) * (a.n_kv * a.group) + w.h * a.group + r % a.group;
                *reinterpret_cast<uint32_t*>(a.out + row * D + d) = pack2(x * inv, y * inv, F16);
            } else {
                *reinterpret_cast<float2*>(piece + r * D + d) = make_float2(x, y);
                if (d == 0) {
                    piece[a.piece_rows * D + r] = m;
                    piece[a.piece_rows * (D + 1) + r] = l;
                }
            }
        }
        if (w.j0 == 0 && w.j1 < w.blocks) {
            cut = true;
            if (threadIdx.x == 0) write_record(a, &w, run.share);
        }
    }
    if (!cut && threadIdx.x == 0) write_record(a, nullptr, run.share);
    if (!ok && lane == 0 && error_flag) atomicExch(error_flag, 1);
}

// Bound by latency: maxima, totals and sums of eight pieces are asked for at once.
constexpr int JOIN_WARPS = 8, JOIN_AHEAD = 8;

// Pieces of attn_few.cu: a warp per row, a lane for D / 32 columns (and for a piece's maximum and total).
template <int D, bool F16>
__device__ __forceinline__ void join_few(const Args& a, int c, int ctas, int q0, int n_rows, int h, int tok0) {
    const int lane = threadIdx.x & 31;
    const int r = blockIdx.y * JOIN_WARPS + (threadIdx.x >> 5);
    if (r >= n_rows) return;
    constexpr int V = D / 32;                                              // columns per lane
    typedef typename std::conditional<V == 4, float4, float2>::type Vec;
    auto piece = [&](int k) { return piece_at<D>(a, c + k, k == 0); };
    float top = -INFINITY, l = 0.f, x[V] = {};
    for (int k0 = 0; k0 < ctas; k0 += 32) {
        const int n = min(32, ctas - k0);
        float m = -INFINITY, t = 0.f;
        if (lane < n) {
            const float* p = piece(k0 + lane);
            m = __ldcg(p + a.piece_rows * D + r);
            t = __ldcg(p + a.piece_rows * (D + 1) + r);
        }
        Vec v[JOIN_AHEAD];
        auto ask = [&](int k) {
#pragma unroll
            for (int i = 0; i < JOIN_AHEAD; ++i)
                if (k + i < n) v[i] = __ldcg(reinterpret_cast<const Vec*>(piece(k0 + k + i) + (int64_t)r * D) + lane);
        };
        ask(0);
        float now = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
        now = fmaxf(now, top);
        const float keep = now == top ? 1.f : ex2(top - now), f = m == -INFINITY ? 0.f : ex2(m - now);
        top = now;
        l = l * keep + warp_sum(f * t);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= keep;
        for (int k = 0; k < n; k += JOIN_AHEAD) {
            if (k > 0) ask(k);
#pragma unroll
            for (int i = 0; i < JOIN_AHEAD; ++i) {
                const float g = __shfl_sync(0xffffffffu, f, (k + i) & 31);
                if (k + i < n) {
                    const float* w = reinterpret_cast<const float*>(&v[i]);
#pragma unroll
                    for (int e = 0; e < V; ++e) x[e] += g * w[e];
                }
            }
        }
    }
    const float inv = top == -INFINITY ? 0.f : 1.f / l;
    const int64_t row = (int64_t)(q0 + tok0 + r / a.group) * (a.n_kv * a.group) + h * a.group + r % a.group;
    uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + row * D + V * lane);
#pragma unroll
    for (int i = 0; i < V; i += 2) dst[i / 2] = pack2(x[i] * inv, x[i + 1] * inv, F16);
}

// Pieces of attn_tiles.cu: CTA y takes rows 32 y .. 32 y + 31, a lane per row and a warp for D / 8 columns; results leave by way of
// shared memory, a row after another.
template <int D, bool F16>
__device__ __forceinline__ void join_tiles(const Args& a, int c, int ctas, int q0, int n_rows, int h, int tok0) {
    constexpr int COLS = D / JOIN_WARPS, PITCH = D / 2 + 4;                // 32-bit words of a row: 16-byte aligned, on other banks than its neighbours
    __shared__ uint32_t rows[32 * PITCH];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = blockIdx.y * 32 + lane;
    if (blockIdx.y * 32 >= n_rows) return;
    const bool valid = r < n_rows;
    auto piece = [&](int k) { return piece_at<D>(a, c + k, k == 0); };
    float top = -INFINITY, l = 0.f, x[COLS] = {};
    for (int k = 0; valid && k < ctas; ++k) {
        const float* p = piece(k);
        const float m = __ldcg(p + D * TILE_ROWS + r), t = __ldcg(p + (D + 1) * TILE_ROWS + r);
        float4 v[COLS / 4];
#pragma unroll
        for (int i = 0; i < COLS / 4; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(p + (warp * COLS + 4 * i) * TILE_ROWS + r * 4));
        const float now = fmaxf(top, m);
        const float keep = now == top ? 1.f : ex2(top - now), f = m == -INFINITY ? 0.f : ex2(m - now);
        top = now;
        l = l * keep + f * t;
#pragma unroll
        for (int i = 0; i < COLS / 4; ++i) {
            x[4 * i] = x[4 * i] * keep + f * v[i].x;
            x[4 * i + 1] = x[4 * i + 1] * keep + f * v[i].y;
            x[4 * i + 2] = x[4 * i + 2] * keep + f * v[i].z;
            x[4 * i + 3] = x[4 * i + 3] * keep + f * v[i].w;
        }
    }
    const float inv = top == -INFINITY ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < COLS; i += 2) rows[lane * PITCH + (warp * COLS + i) / 2] = pack2(x[i] * inv, x[i + 1] * inv, F16);
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * (D / 8); i += 32 * JOIN_WARPS) {
        const int rr = i / (D / 8), d = i % (D / 8), row = blockIdx.y * 32 + rr;
        if (row >= n_rows) break;
        const int64_t at = (int64_t)(q0 + tok0 + row / a.group) * (a.n_kv * a.group) + h * a.group + row % a.group;
        *reinterpret_cast<uint4*>(a.out + at * D + 8 * d) = *reinterpret_cast<const uint4*>(rows + rr * PITCH + 4 * d);
    }
}

// CTA (c, y): of the unit whose first piece is CTA c's, of launch `one`, then of `two`.
template <int D, bool F16>
__global__ void __launch_bounds__(32 * JOIN_WARPS) attn_join_kernel(const __grid_constant__ Args one, const __grid_constant__ Args two, int ctas_of_one) {
    grid_launch_dependents();
    grid_dependency_wait();
    const Args& a = blockIdx.x < ctas_of_one ? one : two;
    const int c = blockIdx.x < ctas_of_one ? blockIdx.x : blockIdx.x - ctas_of_one;
    const int4 rec = __ldcg(reinterpret_cast<const int4*>(a.records + (int64_t)c * RECORD));
    const int ctas = __ldcg(a.records + (int64_t)c * RECORD + 4);
    if (ctas == 0) return;
    const int n_rows = rec.y * a.group;
    if (a.piece_rows == TILE_ROWS) join_tiles<D, F16>(a, c, ctas, rec.x, n_rows, rec.z, rec.w);
    else join_few<D, F16>(a, c, ctas, rec.x, n_rows, rec.z, rec.w);
}

template <int D, bool F16>
int few_launch(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, int ctas, cudaStream_t st) {
    constexpr size_t bytes = sizeof(Shared<D>);
    static SharedLimits limits;
    if (!allow_shared(attn_few_kernel<D, F16>, limits, bytes)) {
        set_error("attention: a CTA cannot have %zu bytes of shared memory", bytes);
        return HQM_ERR_CUDA;
    }
    HQM_CUDA(launch_overlapped(attn_few_kernel<D, F16>, ctas, THREADS, bytes, st, km, vm, a, tc_error_ptr()));
    HQM_LAUNCH_CHECK();
    return HQM_OK;
}

}  // namespace

int launch_few(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, int ctas, int D, bool f16, cudaStream_t st) {
    if (D == 128) return f16 ? few_launch<128, true>(a, km, vm, ctas, st) : few_launch<128, false>(a, km, vm, ctas, st);
    return f16 ? few_launch<64, true>(a, km, vm, ctas, st) : few_launch<64, false>(a, km, vm, ctas, st);
}

int launch_join(const Args& a, const Args* more, int ctas, int D, bool f16, cudaStream_t st) {
    const bool tiles = a.piece_rows == TILE_ROWS;                          // (of two launches that is the first)
    const dim3 grid(more ? 2 * ctas : ctas, tiles ? TILE_ROWS / 32 : FEW_TILE / JOIN_WARPS);
    const Args& b = more ? *more : a;
    if (D == 128) HQM_CUDA(launch_overlapped(f16 ? attn_join_kernel<128, true> : attn_join_kernel<128, false>, grid, 32 * JOIN_WARPS, 0, st, a, b, ctas));
    else HQM_CUDA(launch_overlapped(f16 ? attn_join_kernel<64, true> : attn_join_kernel<64, false>, grid, 32 * JOIN_WARPS, 0, st, a, b, ctas));
    HQM_LAUNCH_CHECK();
    return HQM_OK;
}

}  // namespace attn
}  // namespace hqm
