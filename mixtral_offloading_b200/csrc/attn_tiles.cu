// Attention of many rows per key/value head: prompts, chunks of new tokens, and single tokens beside them, on the
// 5th-generation tensor cores.
//
//     S = Q K^T;  p = 2^(S scale log2 e - m);  O = p V;  l = sum p;  out = O / l
//
// One CTA per SM works through its run of the list of units (attn.cuh).  A unit is 256 rows, two tiles of 128 (row = token *
// group + head), over blocks of 128 positions.  Per block and tile two matrix products of 128 x 128 x D are issued, S into
// tensor memory, and O from p (in tensor memory) and V.  A thread of the four warps of a tile owns one row: maximum, total and
// weights of a row need no other thread.
//
// S does not wait for the weights of the block before: it has columns of its own, and they are free as soon as the tile's warps
// have S in registers.  With D = 64 both tiles have their own, with D = 128 there is room for one S (128 columns of S, 64 of p
// per tile, 128 of O per tile: 512), which the tiles take in turns; each needs it for some 900 of the 3000 cycles that a block's
// weights take.  So the warps that form weights, which set the time, find the next S when they are done with one; where S lay under p
// they waited for both products of their tile in every block, a third of the time.
//
// Bound by the warps that form weights (two per scheduler, 32 x 128 of them in 3000 cycles: 1024 of the special-function unit, 400
// instructions, the latencies between) and, with D = 128, nearly as much by the products: 8000 tokens, 32 on 8 heads, 0.43 ms with 128
// columns (tensor cores 68 %, special-function unit 67 % busy) and 0.42 with 64 (39 %, 67 %).  16001 tokens of 128 columns: 1.84 ms = 1.14
// PFLOP/s, 0.69 of the measured rate of products and 0.82 of the one under the power limit.  Tried and not kept: a part of the
// exponentials by a polynomial on the other units (in this form no gain: 136 us become 146 for 24 packed prompts), 16 warps of half rows,
// blocks of 64 positions, weights formed ahead of their maximum, one warp for both kinds of products (its waits and the
// issues in turn: 2.3 ms), the results of a unit written behind the next one's first weights (5 % slower: registers).
//
// Warps 0-3: weights of tile 0, 4-7: of tile 1, 8: issues the products for S, 11: those for O (an issue takes as long as the product, so
// that one warp for both would leave the tensor cores idle whenever it waits), 9: copies K and V of every block through rings of
// three and two buffers (cp.async.bulk.tensor; of a paged cache a copy per page), 10: walks the list of units and copies their Q.
// K and V have rings of their own, since warp 8 waits for K only and warp 11 for V only (Ring).
//
// The maximum m that a row's weights refer to is raised only when a block exceeds it by more than 2^8: O, which lies in tensor
// memory, is rescaled a few times per unit instead of once per block, weights grow to 256 at the most (of fp16 to 2^15, of which 2^7
// are there to keep small ones: attn.cuh), and l and O mean the same whatever m is.  p is rounded to the type of V, as in attn_few.cuh, with
// the same errors; l adds it before the rounding.
#include <type_traits>

#include "attn_few.cuh"
#include "shared_limit.h"

namespace hqm {
namespace attn {
namespace {

constexpr int KEYS = TILE_KEYS;
constexpr int K_RING = 3, V_RING = 2;
typedef Ring<K_RING> KRing;
typedef Ring<V_RING> VRing;
// Three warpgroups of 168 registers a thread at the launch (64512): the two that form weights take 216, the third keeps 72.
constexpr int WEIGHT_WARPS = 8, THREADS = 32 * WEIGHT_WARPS + 128;
constexpr int REGS_WEIGHTS = 216, REGS_OTHERS = 72;
static_assert(32 * WEIGHT_WARPS * REGS_WEIGHTS + 128 * REGS_OTHERS <= THREADS * 168, "registers of the launch");
constexpr float SLACK = 8.f, LIFT = 7.f;        // (of fp16 weights: 2^15 together)
constexpr int UNIT_EXTRA = 2;         // what a unit costs beside its blocks, in blocks

// A part of a unit (Walk), as the warp that walks the list hands it to the others.
struct Part {
    int tokens;                    // 0: the end of the list
    int q_row, head;               // row of q and out of the first token
    int sees, kv;                  // positions that the first token sees, positions of the sequence
    int j0, j1;                    // blocks
    int end0;                      // blocks j0 .. end0 - 1 hold something that a row of tile 0 sees
    int kv_row, table_row;         // where the sequence begins: packed keys, pages
    int whole;                     // 1: no cut goes through the unit; else 2: its first piece, 0: a later one
};
constexpr int PARTS = 4;

template <int D>
struct Shared {
    static constexpr int HALVES = D / 64;
    static constexpr int PANEL = 128 * 128;                       // 128 rows x 64 columns, 128-byte swizzle
    static constexpr int TILE = HALVES * PANEL;
    alignas(1024) unsigned char q[2][TILE];
    alignas(1024) unsigned char k[K_RING][TILE], v[V_RING][TILE];
    uint64_t k_full[K_RING], k_empty[K_RING], v_full[V_RING], v_empty[V_RING];
    uint64_t q_full[2], q_empty[2], s_full[2], s_read[2], p_full[2], o_done[2];
    uint64_t part_full[PARTS], part_empty[PARTS];
    Part parts[PARTS];
    uint32_t tmem;
};

// Waits until the phase of this parity is over; false (at once from then on) when it has taken about a second.
struct Patience {
    bool ok = true;
    __device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity) {
        const uint32_t at = tc::smem_u32(bar);
        uint32_t done = !ok;
        long long began = 0;
        while (!done) {
            asm volatile(
                "{\n\t.reg .pred p;\n\t"
                "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                "selp.u32 %0, 1, 0, p;\n\t}"
                : "=r"(done) : "r"(at), "r"(parity) : "memory");
            if (!done) {
                const long long now = clock64();
                if (began == 0) began = now;
                else if (now - began > 2000000000ll) { ok = false; return; }
            }
        }
    }
};

__device__ __forceinline__ void expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A lane's row lies in lines of its own, so that the stores of a warp take a cycle per lane and instruction: as wide as they come
// where `out` allows it (Args::out_32), else half of that.
__device__ __forceinline__ void store_32_bytes(void* at, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7]) : "memory");
}

// Two floats for the packed instructions.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float low(Pair v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(Pair v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// The largest; NaN where one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max2(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// V is [position][column]: the product's N runs along a row.  64 columns per 128-byte row; the next 64 a panel further on, the next
// eight positions 1024 bytes.
__device__ __forceinline__ uint64_t desc_across(uint32_t at, int panel) {
    return (uint64_t)((at & 0x3FFFFu) >> 4) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
#define HQM_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define HQM_S8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tmem_load32(uint32_t* r, uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : HQM_R8(r, 0), HQM_R8(r, 8), HQM_R8(r, 16), HQM_R8(r, 24) : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t* r, uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : HQM_R8(r, 0), HQM_R8(r, 8) : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::HQM_S8(r, 0),
                 HQM_S8(r, 8), "r"(at) : "memory");
}
// The loads of r have arrived.  (The registers go through, so that no use of them moves in front.)
#define HQM_B8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void loads_done(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : HQM_B8(r, 0), HQM_B8(r, 8), HQM_B8(r, 16), HQM_B8(r, 24)::"memory");
}
__device__ __forceinline__ void loads_done16(uint32_t* r) { asm volatile("tcgen05.wait::ld.sync.aligned;" : HQM_B8(r, 0), HQM_B8(r, 8)::"memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// True in one lane, the same each time.  (The compiler knows this for one lane: behind `lane == 0` it moved the operands of every
// product into uniform registers one by one, 95 to 125 cycles per instruction instead of 32 or 64.)
__device__ __forceinline__ bool elected() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

__device__ __forceinline__ Cut cut(const Args& a) { return Cut(128 / a.group * 2, TILE_KEYS_LOG, UNIT_EXTRA); }

// What CTA `cta` of `ctas` does.  FIRST: nothing has waited for the grid in front yet.
template <int D, bool F16, bool FIRST>
__device__ __forceinline__ void tiles_cta(Shared<D>& sh, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Args& a, int cta,
                                          int ctas, int* error_flag) {
    using S = Shared<D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_tile = 128 / a.group;                            // tokens
    if (threadIdx.x == 0) {
        for (int i = 0; i < K_RING; ++i) {
            tc::mbar_init(&sh.k_full[i], 1);
            tc::mbar_init(&sh.k_empty[i], 1);
        }
        for (int i = 0; i < V_RING; ++i) {
            tc::mbar_init(&sh.v_full[i], 1);
            tc::mbar_init(&sh.v_empty[i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            tc::mbar_init(&sh.q_full[t], 1);
            tc::mbar_init(&sh.q_empty[t], 1);
            tc::mbar_init(&sh.s_full[t], 1);
            tc::mbar_init(&sh.s_read[t], WEIGHT_WARPS / 2);
            tc::mbar_init(&sh.p_full[t], WEIGHT_WARPS / 2);
            tc::mbar_init(&sh.o_done[t], 1);
        }
        for (int i = 0; i < PARTS; ++i) {
            tc::mbar_init(&sh.part_full[i], 1);
            tc::mbar_init(&sh.part_empty[i], WEIGHT_WARPS + 3);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&qm);
        prefetch_map(&km);
        prefetch_map(&vm);
    }
    if (warp == WEIGHT_WARPS) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&sh.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if constexpr (FIRST) {
        grid_launch_dependents();
        grid_dependency_wait();
    }
    const Cut how = cut(a);
    Run run;
    if (warp == WEIGHT_WARPS + 2) run = find_run(a, how, cta, ctas);       // while tensor memory is allocated
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = sh.tmem;
    Patience patience;
    uint32_t parts = 0;                                            // parts taken
    // The next part; false: there is none.  A warp takes it as a whole, and is done with `sh.parts` when it returns.
    Part w;
    auto next = [&]() {
        const int i = parts % PARTS;
        patience.wait(&sh.part_full[i], (parts / PARTS) & 1);
        ++parts;
        w = sh.parts[i];
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh.part_empty[i]);
        return patience.ok && w.tokens > 0;
    };
    // columns of tensor memory
    constexpr uint32_t S_STEP = D == 64 ? 128 : 0, P_AT = 128 + S_STEP, O_AT = P_AT + 128;
    constexpr int S_COUNT = D == 64 ? 2 : 1;
    if (warp < WEIGHT_WARPS) {
        // ---- weights: thread = row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_WEIGHTS));
        const int t = warp >> 2, r = threadIdx.x & 127;
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);
        const uint32_t s_at = mine + S_STEP * t, p_at = mine + P_AT + 64 * t, o_at = mine + O_AT + D * t;
        const int tok = t * per_tile + r / a.group;                // within the unit
        uint32_t blocks_done = 0;
        while (next()) {
            if (w.tokens <= t * per_tile) continue;
            const bool valid = r < per_tile * a.group && tok < w.tokens;
            const int limit = valid ? min(w.sees + tok, w.kv) : w.kv;          // positions that the row sees
            const int end = t == 0 ? w.end0 : w.j1;
            float m = -INFINITY, l = 0.f;
            for (int j = w.j0; j < end; ++j, ++blocks_done) {
                patience.wait(&sh.s_full[t], blocks_done & 1);
                fence_after();
                uint32_t s[KEYS];
#pragma unroll
                for (int c = 0; c < KEYS; c += 32) tmem_load32(s + c, s_at + c);
#pragma unroll
                for (int c = 0; c < KEYS; c += 32) loads_done(s + c);
                fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh.s_read[S_COUNT == 2 ? t : 0]);
                const int seen = limit - j * KEYS;
                if (__any_sync(0xffffffffu, seen < KEYS)) {
#pragma unroll
                    for (int c = 0; c < KEYS; c += 32)
                        if (__any_sync(0xffffffffu, seen < c + 32)) {
#pragma unroll
                            for (int i = c; i < c + 32; ++i) s[i] = i < seen ? s[i] : 0xff800000u;
                        }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < KEYS; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
                const float block_top = max2(max3(top[0], top[1], top[2]), top[3]) * a.scale_log2;
                const bool raise = valid && !(block_top <= m + (F16 && m < LIFTED_BELOW ? SLACK + LIFT : SLACK));      // (also of NaN)
                if (__any_sync(0xffffffffu, raise)) {
                    float to = max2(m, reference<F16>(block_top, LIFT));
                    if (to == INFINITY) to = NAN;                              // inf - inf, as the definition has it
                    const float f = to == m ? 1.f : ex2(m - to);
                    m = to;
                    l *= f;
                    if (j > w.j0) {
                        patience.wait(&sh.o_done[t], (blocks_done - 1) & 1);
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_load16(o, o_at + c);
                            loads_done16(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_store16(o_at + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : -m;
                const Pair scale2 = pair(a.scale_log2, a.scale_log2), base2 = pair(base, base);
                Pair sum[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < KEYS; c += 32) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const Pair x = fma2(pair(__uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1])), scale2, base2);
                        const Pair y = pair(ex2(low(x)), ex2(high(x)));
                        sum[i & 1] = add2(sum[i & 1], y);
                        p[i] = pack2(low(y), high(y), F16);
                    }
                    if (c == 0 && j > w.j0) {                                  // the product with the weights that lie there is over
                        patience.wait(&sh.o_done[t], (blocks_done - 1) & 1);
                        fence_after();
                    }
                    tmem_store16(p_at + c / 2, p);
                }
                stores_done();
                fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh.p_full[t]);
                sum[0] = add2(sum[0], sum[1]);
                l += low(sum[0]) + high(sum[0]);
            }
            // ---- the part's result ----
            const bool some = w.j0 < end;
            if (some) {
                patience.wait(&sh.o_done[t], (blocks_done - 1) & 1);
                fence_after();
            }
            const bool whole = w.whole == 1;
            const float inv = m == -INFINITY ? 0.f : 1.f / l;
            const int64_t row = ((int64_t)(w.q_row + tok) * a.n_kv + w.head) * a.group + r % a.group;
            const int pr = t * per_tile * a.group + r;
            float* piece = piece_at<D>(a, cta, w.whole >> 1);
            if (valid && !whole) {
                piece[a.piece_rows * D + pr] = m;
                piece[a.piece_rows * (D + 1) + pr] = l;
            }
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tmem_load32(o, o_at + c);
                loads_done(o);
                if (!valid) continue;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = pack2(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv, F16);
                    if (a.out_32) {
                        store_32_bytes(a.out + row * D + c, o);
                        store_32_bytes(a.out + row * D + c + 16, o + 8);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(a.out + row * D + c + 2 * i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(piece + ((c + i) * TILE_ROWS + pr * 4)) =
                            some ? make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]) : make_uint4(0, 0, 0, 0);
                }
            }
            fence_before();
        }
    } else {
        // (A role's code must not come together with one of another number: the compiler counts on the smaller.)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
        if (warp == WEIGHT_WARPS + 1) {
            // ---- copies of K and V ----
            const int rows = a.table ? min(1 << a.page_shift, KEYS) : KEYS;
            const int boxes = KEYS / rows;
            uint32_t at = 0;
            while (next()) {
                const int32_t* table = a.table + (int64_t)w.table_row * a.table_stride;
                for (int j = w.j0; j < w.j1; ++j, ++at) {
                    const int key = j * KEYS + lane * rows;            // of box `lane`; there are eight at the most
                    const int live = min(boxes, (max(w.kv - j * KEYS, 0) + rows - 1) / rows);
                    int row = w.kv_row + key, page = 0;
                    if (a.table && lane < live) {
                        page = min((uint32_t)table[key >> a.page_shift], (uint32_t)a.n_pages);      // outside the pool: zeros
                        row = key & ((1 << a.page_shift) - 1);
                    }
                    auto copy = [&](unsigned char* to, const CUtensorMap* map, uint64_t* full) {
                        patience.ok = __all_sync(0xffffffffu, patience.ok);
                        if (patience.ok) {
                            if (lane == 0) expect(full, (uint32_t)live * rows * 128 * S::HALVES);
                            __syncwarp();
                            if (lane < live)
#pragma unroll
                                for (int h = 0; h < S::HALVES; ++h)
                                    copy_box(tc::smem_u32(to + h * S::PANEL + lane * rows * 128), map, 64 * h, row, w.head, page, full);
                        }
                        __syncwarp();
                    };
                    const int ks = KRing::buffer(at), vs = VRing::buffer(at);
                    if (at >= K_RING) patience.wait(&sh.k_empty[ks], KRing::used(at));
                    copy(sh.k[ks], &km, &sh.k_full[ks]);
                    if (at >= V_RING) patience.wait(&sh.v_empty[vs], VRing::used(at));
                    copy(sh.v[vs], &vm, &sh.v_full[vs]);
                }
            }
            // no copy may be on its way when the CTA ends
            Patience last;
            for (uint32_t k = at < K_RING ? 0 : at - K_RING; k < at; ++k) last.wait(&sh.k_full[KRing::buffer(k)], KRing::copied(k));
            for (uint32_t k = at < V_RING ? 0 : at - V_RING; k < at; ++k) last.wait(&sh.v_full[VRing::buffer(k)], VRing::copied(k));
        } else if (warp == WEIGHT_WARPS) {
            // ---- S = Q K^T ----
            const uint32_t idesc = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((KEYS / 8) << 17) | ((128u >> 4) << 24);
            uint32_t at = 0, units[2] = {0, 0}, made[2] = {0, 0};
            while (next()) {
                for (int j = w.j0; j < w.j1; ++j, ++at) {
                    const int slot = KRing::buffer(at);
                    patience.wait(&sh.k_full[slot], KRing::copied(at));
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int end = t == 0 ? w.end0 : w.tokens > per_tile ? w.j1 : 0;
                        if (j >= end) continue;
                        if (j == w.j0) patience.wait(&sh.q_full[t], units[t]++ & 1);
                        const int buffer = S_COUNT == 2 ? t : 0;
                        if (made[buffer]++ > 0) patience.wait(&sh.s_read[buffer], made[buffer] & 1);       // (of the one before the last)
                        fence_after();
                        if (elected()) {
                            const uint64_t qa = tc::smem_desc_sw128(tc::smem_u32(sh.q[t])), kb = tc::smem_desc_sw128(tc::smem_u32(sh.k[slot]));
#pragma unroll
                            for (int k = 0; k < D / 16; ++k) {
                                const uint64_t off = ((k >> 2) * S::PANEL + (k & 3) * 32) >> 4;
                                mma_ss(tmem + S_STEP * t, qa + off, kb + off, idesc, k > 0);
                            }
                            tc::umma_commit(&sh.s_full[t]);
                            if (j + 1 == end) tc::umma_commit(&sh.q_empty[t]);
                        }
                        __syncwarp();
                    }
                    if (elected()) tc::umma_commit(&sh.k_empty[slot]);
                    __syncwarp();
                }
            }
        } else if (warp == WEIGHT_WARPS + 3) {
            // ---- O += p V ----
            const uint32_t idesc = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (1u << 16) | ((D / 8) << 17) | ((128u >> 4) << 24);
            uint32_t at = 0, used[2] = {0, 0};
            while (next()) {
                for (int j = w.j0; j < w.j1; ++j, ++at) {
                    const int slot = VRing::buffer(at);
                    patience.wait(&sh.v_full[slot], VRing::copied(at));
                    const int live = w.kv - j * KEYS;                      // positions of the block that belong to the sequence
                    if (live < KEYS) {
                        // behind them lies anything, also NaN, which no weight of zero takes away
                        for (int i = max(live, 0) * 8 + lane; i < KEYS * 8; i += 32)
#pragma unroll
                            for (int h = 0; h < S::HALVES; ++h)
                                *reinterpret_cast<uint4*>(sh.v[slot] + h * S::PANEL + i * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (j >= (t == 0 ? w.end0 : w.tokens > per_tile ? w.j1 : 0)) continue;
                        patience.wait(&sh.p_full[t], used[t]++ & 1);
                        fence_after();
                        if (elected()) {
                            const uint64_t vb = desc_across(tc::smem_u32(sh.v[slot]), S::PANEL);
#pragma unroll
                            for (int k = 0; k < KEYS / 16; ++k)
                                mma_ts(tmem + O_AT + D * t, tmem + P_AT + 64 * t + 8 * k, vb + ((k * 16 * 128) >> 4), idesc, j > w.j0 || k > 0);
                            tc::umma_commit(&sh.o_done[t]);
                        }
                        __syncwarp();
                    }
                    if (elected()) tc::umma_commit(&sh.v_empty[slot]);
                    __syncwarp();
                }
            }
        } else {
            // ---- the list, and copies of Q ----
            const uint32_t q_bytes = (uint32_t)(S::HALVES * per_tile * a.group * 128);
            uint32_t copies[2] = {0, 0};
            Walk walk(a, run, how);
            bool split = false, some;
            uint32_t n = 0;
            do {
                some = walk.next();
                if (n >= PARTS) patience.wait(&sh.part_empty[n % PARTS], (n / PARTS - 1) & 1);
                Part p{};
                if (some) {
                    const int tokens = walk.tokens(), sees = walk.s.before + walk.first_token() + 1;
                    const int blocks0 = max(1, (sees + min(per_tile, tokens) - 1 + KEYS - 1) / KEYS);
                    p = Part{tokens, walk.s.q0 + walk.first_token(), walk.h, sees, walk.s.kv, walk.j0, walk.j1, min(blocks0, walk.j1), walk.s.q0, walk.b,
                             walk.whole() ? 1 : 2 * (walk.j0 == 0)};
                }
                if (lane == 0) {
                    sh.parts[n % PARTS] = p;
                    tc::mbar_arrive(&sh.part_full[n % PARTS]);
                }
                __syncwarp();
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (!some || !(t == 0 ? p.j0 < p.end0 : p.tokens > per_tile)) continue;
                    if (copies[t] > 0) patience.wait(&sh.q_empty[t], (copies[t] - 1) & 1);
                    if (!patience.ok) continue;
                    ++copies[t];
                    if (lane == 0) {
                        expect(&sh.q_full[t], q_bytes);
#pragma unroll
                        for (int h = 0; h < S::HALVES; ++h)
                            copy_box(tc::smem_u32(sh.q[t] + h * S::PANEL), &qm, 64 * h, 0, p.head, p.q_row + t * per_tile, &sh.q_full[t]);
                    }
                    __syncwarp();
                }
                if (some && walk.j0 == 0 && walk.j1 < walk.blocks) {
                    split = true;
                    if (lane == 0) write_record(a, &walk, run.share, cta);
                }
                ++n;
            } while (some);
            if (!split && lane == 0) write_record(a, nullptr, run.share, cta);
            Patience last;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (copies[t] > 0) last.wait(&sh.q_full[t], (copies[t] - 1) & 1);
        }
    }
    if (!patience.ok && lane == 0 && error_flag) atomicExch(error_flag, 1);
    fence_before();
    __syncthreads();
    if (warp == WEIGHT_WARPS) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1) attn_tiles_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km,
                                                                const __grid_constant__ CUtensorMap vm, const __grid_constant__ Args a,
                                                                int* error_flag) {
    extern __shared__ __align__(1024) unsigned char raw[];
    tiles_cta<D, F16, true>(*reinterpret_cast<Shared<D>*>(raw), qm, km, vm, a, blockIdx.x, gridDim.x, error_flag);
}

// Single tokens beside chunks: the first CTAs work on the sequences of many rows (a: bound by weights and products), the others on
// those of few (f: bound by the bytes), at the same time.  How many: so that both take as long, from the lengths; a block of 128
// positions and 256 rows is taken for MIXED_COST blocks of 64 positions and few rows.  Two chunks of up to 512 tokens among 30 single
// ones, 32 on 8 heads of 128: 96 us in two launches one after the other; 81, 78, 82 and 96 us with a cost of 2, 3, 4 and 6.  With 64 columns (in
// front of every call the caches are overwritten) 79, 68, 71 and 73 us, for one chunk 77, 66, 65 and 68: the same price for both.
constexpr int MIXED_COST = 3;

template <int D, bool F16>
__global__ void __launch_bounds__(THREADS, 1)
    attn_mixed_kernel(const __grid_constant__ CUtensorMap qm, const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                      const __grid_constant__ CUtensorMap kf, const __grid_constant__ CUtensorMap vf, const __grid_constant__ Args a,
                      const __grid_constant__ Args f, int* error_flag) {
    extern __shared__ __align__(1024) unsigned char raw[];
    __shared__ int64_t cost[2];
    const int warp = threadIdx.x >> 5, cta = blockIdx.x, ctas = gridDim.x;
    grid_launch_dependents();
    grid_dependency_wait();
    if (warp < 2) {
        const int64_t total = warp == 0 ? total_cost(a, cut(a)) * MIXED_COST : total_cost(f, few::cut(f));
        if ((threadIdx.x & 31) == 0) cost[warp] = total;
    }
    __syncthreads();
    const int64_t all = cost[0] + cost[1];
    int first = ctas;                                              // CTAs of the many rows
    if (cost[0] == 0) first = 0;
    else if (cost[1] > 0) first = min(max((int)((float)ctas * (float)cost[0] / (float)all + 0.5f), 1), ctas - 1);
    if (cta < first) {
        if (threadIdx.x == 0) f.records[(int64_t)(ctas - first + cta) * RECORD + 4] = 0;
        tiles_cta<D, F16, false>(*reinterpret_cast<Shared<D>*>(raw), qm, km, vm, a, cta, first, error_flag);
    } else {
        if (threadIdx.x == 0) a.records[(int64_t)cta * RECORD + 4] = 0;
        auto& sh = *reinterpret_cast<few::Shared<D>*>(raw);
        few::begin<D>(sh, kf, vf);
        if (warp == 0) {
            const Run r = find_run(f, few::cut(f), cta - first, ctas - first);
            if (threadIdx.x == 0) sh.run = r;
        }
        __syncthreads();
        if (warp < few::CONSUMERS) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_WEIGHTS));
            few::products<D, F16>(sh, f, cta - first, error_flag);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
            if (warp == few::CONSUMERS) few::copies<D>(sh, kf, vf, f, error_flag);
        }
    }
}
static_assert(few::CONSUMERS == WEIGHT_WARPS && few::THREADS <= THREADS, "attn_mixed_kernel: the warpgroups of both kinds");

template <typename K, typename... A>
int start(K kernel, SharedLimits& limits, size_t bytes, int ctas, cudaStream_t st, const A&... args) {
    if (!allow_shared(kernel, limits, bytes)) {
        set_error("attention: a CTA cannot have %zu bytes of shared memory", bytes);
        return HQM_ERR_CUDA;
    }
    HQM_CUDA(launch_overlapped(kernel, ctas, THREADS, bytes, st, args..., tc_error_ptr()));
    HQM_LAUNCH_CHECK();
    return HQM_OK;
}
template <int D, bool F16>
int tiles_launch(const Args& a, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, int ctas, cudaStream_t st) {
    static SharedLimits limits;
    return start(attn_tiles_kernel<D, F16>, limits, sizeof(Shared<D>), ctas, st, qm, km, vm, a);
}
template <int D, bool F16>
int mixed_launch(const Args& a, const Args& f, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& kf,
                 const CUtensorMap& vf, int ctas, cudaStream_t st) {
    static SharedLimits limits;
    constexpr size_t bytes = sizeof(Shared<D>) > sizeof(few::Shared<D>) ? sizeof(Shared<D>) : sizeof(few::Shared<D>);
    return start(attn_mixed_kernel<D, F16>, limits, bytes, ctas, st, qm, km, vm, kf, vf, a, f);
}

}  // namespace

int launch_tiles(const Args& a, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, int ctas, int D, bool f16, cudaStream_t st) {
    if (D == 128) return f16 ? tiles_launch<128, true>(a, qm, km, vm, ctas, st) : tiles_launch<128, false>(a, qm, km, vm, ctas, st);
    return f16 ? tiles_launch<64, true>(a, qm, km, vm, ctas, st) : tiles_launch<64, false>(a, qm, km, vm, ctas, st);
}

int launch_mixed(const Args& a, const Args& f, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& kf,
                 const CUtensorMap& vf, int ctas, int D, bool f16, cudaStream_t st) {
    if (D == 128) return f16 ? mixed_launch<128, true>(a, f, qm, km, vm, kf, vf, ctas, st) : mixed_launch<128, false>(a, f, qm, km, vm, kf, vf, ctas, st);
    return f16 ? mixed_launch<64, true>(a, f, qm, km, vm, kf, vf, ctas, st) : mixed_launch<64, false>(a, f, qm, km, vm, kf, vf, ctas, st);
}

}  // namespace attn
}  // namespace hqm
