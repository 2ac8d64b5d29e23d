// What the attention kernels over new tokens share: their arguments, how the work is cut, and the partial results.
//
// A launch covers sequences of different lengths: sequence b has n_b new tokens (rows cu[b] .. cu[b + 1] of q) and L_b
// positions of keys and values, the new ones last; new token i sees positions 0 .. L_b - n_b + i.  The `group` query heads of one
// key/value head are rows of the same tile (row = token * group + head), so that keys and values are read once for all of them.
//
// The work is a list of units (sequence, key/value head, tile of rows), each of as many blocks of keys as its last row sees, at
// least one.  The list is cut into runs of equal cost, one per CTA, wherever that falls; a unit costs its blocks and, in front of
// them, `extra` blocks for its beginning and end (a cut in there falls in front of the unit).  Every CTA finds its run from
// the lengths in device memory, so the host needs no length and a captured graph follows them.  A unit that a cut goes through leaves
// unnormalised sums with their maximum and total (a "piece") per CTA, which attn_join adds in the order of the CTAs: the same
// bits for the same lengths, whichever CTA ends first.
#pragma once
#include <cuda.h>

#include "common.cuh"
#include "kernels.cuh"

namespace hqm {
namespace attn {

struct Args {
    const uint16_t* q;
    uint16_t* out;                 // (T, n_heads, D), contiguous
    int out_32;                    // whether out begins on a 32-byte boundary (a 16-byte one it does in any case)
    int64_t q_token, q_head;       // strides of q, in elements
    const int32_t* table;          // null: keys and values are packed like the queries
    int64_t table_stride;
    const int32_t* cu;             // B + 1
    const int32_t* kv_lens;        // null with table
    int B, T, n_kv, group;
    int n_pages, max_pages, page_shift;
    float scale_log2;              // softmax scale times log2(e)
    float* pieces;                 // two per CTA
    int32_t* records;              // of CTA c: the unit that starts in c and is cut behind it (RECORD words)
    int piece_rows;                // rows of a piece
    int rows_above, rows_upto;     // the launch is about sequences with that many rows per key/value head
    int cuts;                      // 0: a CTA takes the units that begin in its run as a whole, and there is nothing to join
};
constexpr int RECORD = 8;          // q0, tokens, head, first token, CTAs (0: none), 3 unused

// a / b for a >= 0, b > 0.  (A division of 64 bits is a routine of some 600 cycles.)
__host__ __device__ inline int64_t quotient(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// Sum of floor((a i + b) / m) over i = 0 .. n - 1 (the sum of an arithmetic progression per step of Euclid's algorithm on a, m).
__host__ __device__ inline int64_t floor_sum(int64_t n, uint32_t m, uint32_t a, uint32_t b) {
    int64_t sum = 0;
    while (n > 0) {
        if (a >= m) { sum += (n - 1) * n / 2 * (a / m); a %= m; }
        if (b >= m) { sum += n * (b / m); b %= m; }
        const int64_t y = (int64_t)a * n + b;
        if (y < m) break;
        n = quotient(y, m);
        b = (uint32_t)(y - n * m);
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// How a kernel cuts the work.
struct Cut {
    int per, block_log, extra;     // tokens per tile, log2 of the keys per block, blocks that a unit costs beside its own
    int per_log;                   // log2 of per, -1 where it is not a power of two
    __host__ __device__ Cut(int per_, int block_log_, int extra_) : per(per_), block_log(block_log_), extra(extra_), per_log(-1) {
        if ((per & (per - 1)) == 0)
            for (per_log = 0; (1 << per_log) < per; ++per_log) {}
    }
    __host__ __device__ int tiles(int n) const {           // of n tokens
        const uint32_t up = (uint32_t)n + per - 1;
        return (int)(per_log >= 0 ? up >> per_log : up / (uint32_t)per);
    }
};

// One sequence's part of the list.
struct Seq {
    int q0, n;                     // rows of q
    int kv;                        // positions that can be read
    int before;                    // kv - n: what token 0 sees, less one
    int tiles;                     // tiles of rows
    __host__ __device__ int blocks(const Cut& c, int tile) const {
        const int seen = before + min((tile + 1) * c.per, n);
        return max(1, (seen + (1 << c.block_log) - 1) >> c.block_log);
    }
    // Cost of tiles 0 .. count - 1.  A tile that sees nothing has one block.  The others of `per` tokens, from tile `empty` on, have
    // floor((per i + b) / block): where both are powers of two the sum is that of an arithmetic progression in groups of equal terms.
    // Nothing where the launch leaves the sequence out (tiles == 0), also where it has fewer positions than tokens: a walk passes it
    // without a cost, and runs that did not agree with that would leave blocks to nobody.
    __host__ __device__ int64_t prefix(const Cut& c, int count) const {
        if (tiles == 0) return 0;
        const int whole = min(count, tiles - 1);               // tiles of `per` tokens
        int empty = 0;
        if (before < 0) empty = min(whole, -before / c.per);
        int64_t sum = (int64_t)count * c.extra + empty;
        if (whole > empty) {
            const int64_t n = whole - empty;
            const uint32_t b = (uint32_t)((int64_t)before + (int64_t)(empty + 1) * c.per + (1 << c.block_log) - 1);
            if (c.per_log < 0) sum += floor_sum(n, 1u << c.block_log, c.per, b);
            else if (c.per_log >= c.block_log) sum += (n * (n - 1) / 2 << (c.per_log - c.block_log)) + n * (b >> c.block_log);
            else {
                const int k = c.block_log - c.per_log;         // 2^k tiles of equal blocks
                auto upto = [k](int64_t x) { const int64_t y = x >> k; return (y * (y - 1) / 2 << k) + (x - (y << k)) * y; };
                const int64_t first = b >> c.per_log;
                sum += upto(first + n) - upto(first);
            }
        }
        if (count >= tiles) sum += blocks(c, tiles - 1);
        return sum;
    }
};

__host__ __device__ __forceinline__ Seq load_seq(const Args& a, int b, const Cut& c) {
    Seq s;
    const int lo = min(max(a.cu[b], 0), a.T), hi = min(max(a.cu[b + 1], lo), a.T);
    s.q0 = lo;
    s.n = hi - lo;
    s.kv = s.n;
    if (a.table) s.kv = (int)min((int64_t)max(a.kv_lens[b], 0), (int64_t)a.max_pages << a.page_shift);
    s.before = s.kv - s.n;
    const int64_t rows = (int64_t)s.n * a.group;
    s.tiles = rows > a.rows_above && rows <= a.rows_upto ? c.tiles(s.n) : 0;
    return s;
}

// Where a CTA's run of blocks begins, and how long it is.
struct Run {
    int64_t share;                 // cost of every run (the last one may have less)
    int64_t left;                  // of this one
    int b, h, tile;
    int skip;                      // cost of its first unit that lies in front of the run
    Seq s;                         // sequence b
};

// Cost of the whole list.  Called by one whole warp.
__device__ inline int64_t total_cost(const Args& a, const Cut& c) {
    int64_t total = 0;
#pragma unroll 1
    for (int b = threadIdx.x & 31; b < a.B; b += 32) {
        const Seq s = load_seq(a, b, c);
        total += s.prefix(c, s.tiles);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    return total * a.n_kv;
}

// Called by one whole warp; every lane gets the run of CTA `cta` of `ctas`.
__device__ inline Run find_run(const Args& a, const Cut& c, int cta, int ctas) {
    const int lane = threadIdx.x & 31;
    auto cost = [&](const Seq& s) { return s.prefix(c, s.tiles) * a.n_kv; };
    auto upto = [&](int64_t w) {                               // sum over the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += v;
        }
        return w;
    };
    // a lane's share of the sequences, in one stretch; then the stretch that the run begins in, a sequence per lane
    const int stretch = (a.B + 31) / 32;
    Seq mine{};
    int64_t w = 0;
#pragma unroll 1
    for (int i = 0; i < stretch; ++i) {
        const int b = lane * stretch + i;
        if (b >= a.B) break;
        mine = load_seq(a, b, c);
        w += cost(mine);
    }
    int64_t sum = upto(w);
    const int64_t total = __shfl_sync(0xffffffffu, sum, 31);
    Run r;
    r.share = quotient(total + ctas - 1, ctas);
    const int64_t lo = r.share * cta;
    r.left = min(max(total - lo, (int64_t)0), r.share);
    r.b = r.h = r.tile = r.skip = 0;
    if (r.left == 0) return r;
    const int owner = __ffs(__ballot_sync(0xffffffffu, sum > lo)) - 1;
    int64_t base = stretch == 1 ? 0 : __shfl_sync(0xffffffffu, sum - w, owner);
    const int from = stretch == 1 ? 0 : owner * stretch, to = stretch == 1 ? a.B : min(from + stretch, a.B);
    for (int b0 = from; b0 < to; b0 += 32) {
        if (stretch > 1) {
            mine = Seq{};
            if (b0 + lane < to) mine = load_seq(a, b0 + lane, c);
            w = cost(mine);
            sum = upto(w);
        }
        const uint32_t past = __ballot_sync(0xffffffffu, base + sum > lo);
        if (past) {
            const int src = __ffs(past) - 1;
            r.b = b0 + src;
            const int64_t off = lo - (base + __shfl_sync(0xffffffffu, sum - w, src));
            Seq& s = r.s;
            s.q0 = __shfl_sync(0xffffffffu, mine.q0, src);
            s.n = __shfl_sync(0xffffffffu, mine.n, src);
            s.kv = __shfl_sync(0xffffffffu, mine.kv, src);
            s.before = s.kv - s.n;
            s.tiles = c.tiles(s.n);
            const int64_t one = quotient(__shfl_sync(0xffffffffu, w, src), a.n_kv);
            r.h = (int)quotient(off, one);
            const int64_t in = off - r.h * one;
            // the last tile whose prefix is <= in: of t0 .. t0 + n - 1, 32 places in between at a time
            int t0 = 0, n = s.tiles;
            int64_t before = 0;                                // prefix(t0)
            while (n > 1) {
                const int step = (n + 31) / 32, t = t0 + lane * step;
                const int64_t p = lane * step < n ? s.prefix(c, t) : INT64_MAX;
                const int at = 31 - __clz(__ballot_sync(0xffffffffu, p <= in));
                before = __shfl_sync(0xffffffffu, p, at);
                t0 += at * step;
                n = min(step, n - at * step);
            }
            r.tile = t0;
            r.skip = (int)(in - before);
            return r;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    r.left = 0;
    return r;
}

// A CTA's walk through its run: every part of a unit that it works on, in order.  All threads that walk it see the same.
struct Walk {
    const Args& a;
    Cut cut;
    Seq s;
    int64_t left;
    int b, h, tile, skip;
    int j0, j1, blocks;            // the part: blocks j0 .. j1 - 1 of `blocks`
    __host__ __device__ Walk(const Args& args, const Run& r, const Cut& c) : a(args), cut(c), s(r.s), left(r.left), b(r.b), h(r.h), tile(r.tile), skip(r.skip) {}
    __host__ __device__ bool next() {      // false: done
        while (left > 0) {
            if (tile == s.tiles) {
                tile = 0;
                if (++h == a.n_kv) {
                    h = 0;
                    do s = load_seq(a, ++b, cut);
                    while (s.tiles == 0);
                }
            }
            blocks = s.blocks(cut, tile++);
            if (!a.cuts) {
                const bool begins = skip == 0;
                left -= blocks + cut.extra - skip;
                skip = 0;
                j0 = 0;
                j1 = blocks;
                if (begins) return true;
                continue;
            }
            const int end = (int)min((int64_t)(blocks + cut.extra), skip + left);
            left -= end - skip;
            j0 = max(skip - cut.extra, 0);
            j1 = max(end - cut.extra, 0);
            skip = 0;
            if (j1 > j0) return true;
        }
        return false;
    }
    // the part's tile is tile - 1 from here on
    __host__ __device__ int first_token() const { return (tile - 1) * cut.per; }
    __host__ __device__ int tokens() const { return min(cut.per, s.n - first_token()); }
    __host__ __device__ bool whole() const { return j0 == 0 && j1 == blocks; }
};

// A piece: sums, then maxima [rows] (base 2), then totals [rows].  The sums of attn_few.cu lie as [rows][D]; those of attn_tiles.cu, where
// neighbouring lanes hold neighbouring rows, as [D / 4][rows][4], so that a warp's store is one stretch.
template <int D>
__device__ __forceinline__ float* piece_at(const Args& a, int cta, int tail) {
    return a.pieces + (int64_t)(2 * cta + tail) * a.piece_rows * (D + 2);
}
inline size_t piece_bytes(int ctas, int rows, int D) { return (size_t)2 * ctas * rows * (D + 2) * sizeof(float); }
inline size_t record_bytes(int ctas) { return ((size_t)ctas * RECORD * sizeof(int32_t) + 255) / 256 * 256; }

// CTA c's record: about the unit that its run ends in the middle of and that began in it, if there is one.
__device__ __forceinline__ void write_record(const Args& a, const Walk* w, int64_t share, int cta) {
    int32_t* r = a.records + (int64_t)cta * RECORD;
    if (!w) {
        r[4] = 0;
        return;
    }
    r[0] = w->s.q0;
    r[1] = w->tokens();
    r[2] = w->h;
    r[3] = w->first_token();
    r[4] = 1 + (int)quotient(w->blocks - w->j1 + share - 1, share);      // this CTA and those that the rest reaches into
}

__device__ __forceinline__ uint16_t to_bits(float v, bool f16) {
    return f16 ? __half_as_ushort(__float2half_rn(v)) : float_to_bf16_bits(v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool f16) {      // lo in the lower half
    uint32_t r;
    if (f16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// What the weights 2^(x - reference) of a row refer to, from its largest x.  fp16 ends at 2^-24: where the largest weight were 1, a key 17
// below the largest in e's powers would count in the total and not in the sum with v, 0.4 % of a row with 130000 of them.  So the
// reference is `lift` lower, the largest weight 2^lift, and maxima, totals and sums of pieces mean that reference.  Not from 2^19 on, where
// x is known to 2^-5 and worse and the largest weight has to stay clear of 65504.
constexpr float LIFTED_BELOW = 524288.f;
template <bool F16>
__device__ __forceinline__ float reference(float top, float lift) {
    return F16 && top < LIFTED_BELOW ? top - lift : top;
}

// Adds the pieces of the units that a cut goes through, of one launch or of two (attn_few.cu).
int launch_join(const Args& a, const Args* more, int ctas, int D, bool f16, cudaStream_t st);
// attn_few.cu: up to FEW_TILE rows per key/value head.
int launch_few(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, int ctas, int D, bool f16, cudaStream_t st);

// attn_tiles.cu: any number.
int launch_tiles(const Args& a, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, int ctas, int D, bool f16, cudaStream_t st);
// Both at once, f about the sequences of few rows.
int launch_mixed(const Args& a, const Args& f, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& kf,
                 const CUtensorMap& vf, int ctas, int D, bool f16, cudaStream_t st);

// A ring of N buffers with a barrier for "copied" and one for "used" each; item i of a warp's list lies in buffer(i).  A barrier tells the
// phase that it is in by its parity alone, so a warp that waits on one has to wait for every phase of it, one after another: for a
// phase whose predecessor it has not seen a wait passes at once, on what lay there before.  Hence every warp that waits
// on a ring takes all of its items.
template <int N>
struct Ring {
    __host__ __device__ static int buffer(uint32_t i) { return (int)(i % N); }
    __host__ __device__ static uint32_t copied(uint32_t i) { return (i / N) & 1; }             // parity of the phase in which item i arrives
    __host__ __device__ static uint32_t used(uint32_t i) { return (i / N - 1) & 1; }           // in which the item in its place before was used, i >= N
};

constexpr int FEW_TILE = 16;       // rows of a unit of attn_few.cu
constexpr int FEW_KEYS = 64, FEW_KEYS_LOG = 6;         // positions of a block there
constexpr int TILE_ROWS = 256;     // rows of a unit of attn_tiles.cu
constexpr int TILE_KEYS = 128, TILE_KEYS_LOG = 7;      // positions of a block there
constexpr int MIXED_ROWS = 64;     // see attn.cu
constexpr int FEW_WHOLE = 5, TILES_WHOLE = 4;              // blocks, see attn.cu
constexpr int MAX_GROUP = 128;     // query heads per key/value head: the rows of a tile

}  // namespace attn
}  // namespace hqm
