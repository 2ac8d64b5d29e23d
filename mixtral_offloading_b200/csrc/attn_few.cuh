// Attention of a few rows per key/value head (single tokens, short continuations) over pages of keys and values: what a CTA does.
//
//     out = softmax(q k^T scale) v,   2^(x log2 e) for exp, running maximum and total per row
//
// Bound by the bytes of keys and values: 4 D per position and key/value head.  One CTA per SM; a warp keeps a ring of stages
// full with tiled copies (64 positions of K and V each), eight warps work on them, two stages at a time, sixteen positions per
// warp.  Each warp has its own running maximum, total and sums, so that nothing is exchanged before the end of a unit.  The
// products go through mma.sync m16n8k16: with 16 rows at the most the matrix unit of tcgen05 would work on 128 rows of which
// seven eighths are padding, and the bytes, not the products, set the time.  64 tokens behind 4970 positions on average, 32 on 8
// heads of 128: 207 us = 6.29 TB/s, 0.96 of a plain copy's rate; one token behind 130001 positions: 93 us, 5.7 TB/s, the rest is
// start-up and the join.  A CTA's own work takes 450 cycles per block of 64 positions, its share of the memory's rate 1200.  Six
// stages instead of four changed nothing.
//
// Weights are rounded to the type of V, which the product takes for both operands: half a step of each, so that errors against 64 bits are
// 1.1 to 1.4 times those of 32-bit weights (0.0021 and 0.0017 of the result with bf16, whose own rounding is most of either).  Their total
// is formed before the rounding, in fp32 as everything else.
#pragma once
#include <type_traits>

#include "attn.cuh"
#include "tc_common.cuh"

namespace hqm {
namespace attn {
namespace few {

constexpr int CONSUMERS = 8;
constexpr int THREADS = 32 * (CONSUMERS + 1);
constexpr int STAGES = 4;
static_assert(STAGES % 2 == 0, "the halves of the warps take turns: a buffer belongs to one half, or that one would skip every other phase");
constexpr int UNIT_EXTRA = 1;          // what a unit costs beside its blocks, in blocks
constexpr float LIFT = 15.f;           // of fp16 weights (attn.cuh): up to 2^15

template <int D>
struct Shared {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = FEW_KEYS * 128 * HALVES;          // 64 positions: boxes of [64 columns][rows of a box][128 bytes], 128-byte swizzle
    alignas(1024) unsigned char ring[STAGES][2][TILE];            // K, V
    static constexpr int PITCH = D + 8;                           // four rows of a quad's eight columns on banks of their own
    float sums[CONSUMERS][FEW_TILE][PITCH];
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

__device__ __forceinline__ Cut cut(const Args& a) { return Cut(FEW_TILE / a.group, FEW_KEYS_LOG, UNIT_EXTRA); }

// In front of grid_dependency_wait().
template <int D>
__device__ __forceinline__ void begin(Shared<D>& sh, const CUtensorMap& km, const CUtensorMap& vm) {
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            tc::mbar_init(&sh.full[i], 1);
            tc::mbar_init(&sh.empty[i], CONSUMERS / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&km);
        prefetch_map(&vm);
    }
}

// Warp CONSUMERS: the copies, lane i brings box i of a stage, K and V.
template <int D>
__device__ __forceinline__ void copies(Shared<D>& sh, const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int* error_flag) {
    using S = Shared<D>;
    const int lane = threadIdx.x & 31;
    Walk w(a, sh.run, cut(a));
    bool ok = true;
    const int rows_log = a.table ? min(a.page_shift, FEW_KEYS_LOG) : FEW_KEYS_LOG, rows = 1 << rows_log;         // of a box
    const int boxes_log = FEW_KEYS_LOG - rows_log, boxes = 1 << boxes_log;                                     // per block
    {
        uint32_t at = 0;
        while (w.next() && ok) {
            const int32_t* table = a.table + (int64_t)w.b * a.table_stride;
            // Entries of the table, 32 at once and a round ahead of the copies (one that waits for its entry takes some 800 cycles; 130001
            // positions: 98 us when an entry was read one block ahead, 93 so): lane i has that of box i % boxes of block from + i / boxes.
            auto entries = [&](int from) {
                const int j = from + (lane >> boxes_log), key = j * FEW_KEYS + (lane & (boxes - 1)) * rows;
                if (!a.table || j >= w.j1 || key >= w.s.kv) return 0;
                return (int)min((uint32_t)table[key >> a.page_shift], (uint32_t)a.n_pages);      // outside the pool: zeros
            };
            const int round = 32 >> boxes_log;
            int now = 0, ahead = entries(w.j0);
            for (int j = w.j0; j < w.j1 && ok; ++j, ++at) {
                const int in = (j - w.j0) & (round - 1);
                if (in == 0) {
                    now = ahead;
                    ahead = entries(j + round);
                }
                const int page = __shfl_sync(0xffffffffu, now, (in * boxes + lane) & 31);
                const int key = j * FEW_KEYS + lane * rows, row = a.table ? key & ((1 << a.page_shift) - 1) : w.s.q0 + key;
                const int stage = at % STAGES;
                if (at >= STAGES) ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh.empty[stage], (at / STAGES - 1) & 1));
                if (!ok) break;
                const int live = min(boxes, (max(w.s.kv - j * FEW_KEYS, 0) + rows - 1) >> rows_log);  // boxes that hold positions of the sequence
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
    }
}

// Warps 0 .. CONSUMERS - 1: the products.
template <int D, bool F16>
__device__ __forceinline__ void products(Shared<D>& sh, const Args& a, int cta, int* error_flag) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Run& run = sh.run;
    Walk w(a, run, cut(a));
    bool ok = true;
    const int rows = a.table ? min(1 << a.page_shift, FEW_KEYS) : FEW_KEYS;
    const int half = warp >> 2, strip = (warp & 3) * 16;                   // stages of this half, positions within a stage
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;                         // rows r0 and r0 + 8, columns c0, c0 + 1 of an 8-wide tile
    // where position `key` of a stage lies, its first 64 columns; the next 64 are `across` bytes further on
    auto key_at = [&](int key) { return (uint32_t)(((key & ~(rows - 1)) * (D / 64) + (key & (rows - 1))) * 128); };
    const int across = rows * 128;
    const int krow = strip + (lane & 7) + ((lane >> 4) << 3), kch = (lane >> 3) & 1, vrow = strip + (lane & 15), vch = lane >> 4;
    // (16-byte columns of a row lie at their number xor the row's: those of step k at the first step's address xor 32 k)
    const uint32_t k_off = key_at(krow) + ((kch ^ (krow & 7)) << 4), v_off = key_at(vrow) + ((vch ^ (vrow & 7)) << 4);
    int tok[2];                                                            // of the two rows: token within the unit, where its q lies
    int64_t q_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        tok[i] = (r0 + 8 * i) / a.group;
        q_at[i] = tok[i] * a.q_token + (r0 + 8 * i - tok[i] * a.group) * a.q_head + c0;
    }
    // of the row that this thread writes results of, the first of its n_rows * D / 2 / threads
    const int out_row = threadIdx.x / (D / 2), out_step = 32 * CONSUMERS / (D / 2);
    uint32_t at = 0;
    bool split = false;
    while (w.next()) {
        const int tok0 = w.first_token(), n_rows = w.tokens() * a.group;
        uint32_t qf[D / 16][4];
        int limit[2];                                                      // positions that the two rows see
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool valid = r0 + 8 * i < n_rows;
            limit[i] = valid ? w.s.before + tok0 + tok[i] + 1 : w.s.kv;    // (a row of padding is nobody's)
            const uint16_t* src = a.q + (int64_t)(w.s.q0 + tok0) * a.q_token + (int64_t)(w.h * a.group) * a.q_head + q_at[i];
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qf[k][i] = valid ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
                qf[k][i + 2] = valid ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
            }
            if (valid && w.h + 1 < a.n_kv && (lane & 3) < D / 64)          // the next unit's, most of the time
                asm volatile("prefetch.global.L1 [%0];" ::"l"(src + a.group * a.q_head + (lane & 3) * 64));
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
                float s[2][4] = {}, s2[2][4] = {};                         // two sums each, so that half as many products wait for one another
#pragma unroll
                for (int k = 0; k < D / 16; k += 2) {
                    uint32_t b[4], b2[4];
                    const uint32_t from = kt + (k >> 2) * across;
                    ldsm(b, from ^ ((k & 3) << 5));
                    ldsm(b2, from ^ (((k + 1) & 3) << 5));
                    mma<F16>(s[0], qf[k], b[0], b[1]);
                    mma<F16>(s[1], qf[k], b[2], b[3]);
                    mma<F16>(s2[0], qf[k + 1], b2[0], b2[1]);
                    mma<F16>(s2[1], qf[k + 1], b2[2], b2[3]);
                }
                float now[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][e] += s2[t][e];
                if (__any_sync(0xffffffffu, min(limit[0], limit[1]) < key0 + 16)) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (key0 + 8 * t + c0 + (e & 1) >= limit[e >> 1]) s[t][e] = -INFINITY;
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) now[e >> 1] = fmaxf(now[e >> 1], s[t][e]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 1));
                    now[i] = fmaxf(now[i], __shfl_xor_sync(0xffffffffu, now[i], 2));
                    now[i] = fmaxf(reference<F16>(now[i] * a.scale_log2, LIFT), top[i]);
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
                const float base[2] = {top[0] == -INFINITY ? 0.f : -top[0], top[1] == -INFINITY ? 0.f : -top[1]};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[t][e] = ex2(fmaf(s[t][e], a.scale_log2, base[e >> 1]));
                        total[e >> 1] += s[t][e];
                    }
                const uint32_t p[4] = {pack2(s[0][0], s[0][1], F16), pack2(s[0][2], s[0][3], F16), pack2(s[1][0], s[1][1], F16),
                                       pack2(s[1][2], s[1][3], F16)};
                auto add = [&](auto masked, uint32_t m0, uint32_t m1) {
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        uint32_t b[4];
                        ldsm_t(b, (vt + (d >> 2) * across) ^ ((d & 3) << 5));
                        if constexpr (decltype(masked)::value) {
                            b[0] &= m0, b[2] &= m0;
                            b[1] &= m1, b[3] &= m1;
                        }
                        mma<F16>(o[2 * d], p, b[0], b[1]);
                        mma<F16>(o[2 * d + 1], p, b[2], b[3]);
                    }
                };
                if (key0 + 16 <= w.s.kv) add(std::false_type{}, 0u, 0u);
                else {
                    // what lies behind the sequence is anything, also NaN, which no weight of zero takes away
                    const int k0 = key0 + c0;
                    add(std::true_type{}, (k0 < w.s.kv ? 0xffffu : 0u) | (k0 + 1 < w.s.kv ? 0xffff0000u : 0u),
                        (k0 + 8 < w.s.kv ? 0xffffu : 0u) | (k0 + 9 < w.s.kv ? 0xffff0000u : 0u));
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
        float* piece = whole ? nullptr : piece_at<D>(a, cta, w.j0 == 0);
        const int64_t row0 = (int64_t)(w.s.q0 + tok0) * (a.n_kv * a.group) + w.h * a.group;
        for (int r = out_row; r < n_rows; r += out_step) {
            const int d = threadIdx.x % (D / 2) * 2;
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
                const int64_t row = row0 + r + (n_rows > a.group ? r / a.group * (a.n_kv - 1) * a.group : 0);
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
            split = true;
            if (threadIdx.x == 0) write_record(a, &w, run.share, cta);
        }
    }
    if (!split && threadIdx.x == 0) write_record(a, nullptr, run.share, cta);
    if (!ok && lane == 0 && error_flag) atomicExch(error_flag, 1);
}

}  // namespace few
}  // namespace attn
}  // namespace hqm
