// Attention of a few rows per key/value head (attn_few.cuh), and the pass that joins pieces of cut units for every attention kernel
// of the library.
#include <type_traits>

#include "attn_few.cuh"
#include "shared_limit.h"

namespace hqm {
namespace attn {
namespace {

template <int D, bool F16>
__global__ void __launch_bounds__(few::THREADS, 1) attn_few_kernel(const __grid_constant__ CUtensorMap km, const __grid_constant__ CUtensorMap vm,
                                                                   const __grid_constant__ Args a, int* error_flag) {
    extern __shared__ __align__(1024) unsigned char raw[];
    auto& sh = *reinterpret_cast<few::Shared<D>*>(raw);
    few::begin<D>(sh, km, vm);
    grid_launch_dependents();
    grid_dependency_wait();
    if (threadIdx.x < 32) {
        const Run r = find_run(a, few::cut(a), blockIdx.x, gridDim.x);
        if (threadIdx.x == 0) sh.run = r;
    }
    __syncthreads();
    if (threadIdx.x >= 32 * few::CONSUMERS) few::copies<D>(sh, km, vm, a, error_flag);
    else few::products<D, F16>(sh, a, blockIdx.x, error_flag);
}

// Bound by latency (4 to 6 us): maxima, totals and sums of up to eight pieces are asked for at once.
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
    float ms[2], ts[2];
    float4 vs[2][COLS / 4];
    auto ask = [&](int k, int s) {                                         // the next piece, while one is added
        const float* p = piece(k);
        ms[s] = __ldcg(p + D * TILE_ROWS + r);
        ts[s] = __ldcg(p + (D + 1) * TILE_ROWS + r);
#pragma unroll
        for (int i = 0; i < COLS / 4; ++i) vs[s][i] = __ldcg(reinterpret_cast<const float4*>(p + (warp * COLS + 4 * i) * TILE_ROWS + r * 4));
    };
    auto add = [&](int s) {
        const float m = ms[s], t = ts[s];
        const float4* v = vs[s];
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
    };
    if (valid) {
        ask(0, 0);
        for (int k = 0; k < ctas; k += 2) {
            if (k + 1 < ctas) ask(k + 1, 1);
            add(0);
            if (k + 2 < ctas) ask(k + 2, 0);
            if (k + 1 < ctas) add(1);
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
    constexpr size_t bytes = sizeof(few::Shared<D>);
    static SharedLimits limits;
    if (!allow_shared(attn_few_kernel<D, F16>, limits, bytes)) {
        set_error("attention: a CTA cannot have %zu bytes of shared memory", bytes);
        return HQM_ERR_CUDA;
    }
    HQM_CUDA(launch_overlapped(attn_few_kernel<D, F16>, ctas, few::THREADS, bytes, st, km, vm, a, tc_error_ptr()));
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
