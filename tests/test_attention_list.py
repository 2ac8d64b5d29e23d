"""The list of units that the attention kernels cut into runs (csrc/attn.cuh), walked on the host: costs do not fall from tile to tile,
and the runs of all CTAs cover every block of every unit once, whatever the lengths are and whichever sequences a launch leaves
to the other kernel."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

SOURCE = r"""
#include "attn.cuh"
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>
using namespace hqm::attn;

static int failures = 0;
#define EXPECT(cond, ...) do { if (!(cond) && failures++ < 20) { printf(__VA_ARGS__); printf("\n"); } } while (0)

static void walk_all(const std::vector<int>& n, const std::vector<int>& L, int group, int n_kv, const Cut& c, int above, int upto, int ctas, int cuts) {
    const int B = (int)n.size();
    std::vector<int32_t> cu{0}, lens(L);
    for (int v : n) cu.push_back(cu.back() + v);
    Args a{};
    const int32_t some = 0;
    a.table = &some;                                                   // pages: lengths from kv_lens
    a.B = B, a.T = cu.back(), a.n_kv = n_kv, a.group = group, a.max_pages = 1 << 20, a.page_shift = 4, a.rows_above = above, a.rows_upto = upto, a.cuts = cuts;
    cu.push_back(a.T + 100000), lens.push_back(100000);                // behind the list: a walk that gets there is seen
    a.T += 100000;
    a.cu = cu.data(), a.kv_lens = lens.data();
    int64_t total = 0;
    std::vector<int64_t> first;                                        // cost in front of a sequence
    for (int b = 0; b < B; ++b) {
        const Seq s = load_seq(a, b, c);
        const int64_t rows = (int64_t)n[b] * group;
        EXPECT(s.tiles == (rows > above && rows <= upto ? c.tiles(n[b]) : 0), "sequence %d: %d tiles", b, s.tiles);
        int64_t before = 0, plain = 0;
        for (int t = 0; t <= s.tiles; ++t) {
            const int64_t p = s.prefix(c, t);
            EXPECT(p >= before, "new %d, positions %d: cost %lld of %d tiles, %lld of one less", n[b], lens[b], (long long)p, t, (long long)before);
            EXPECT(p == plain, "new %d, positions %d: cost %lld of %d tiles, %lld one by one", n[b], lens[b], (long long)p, t, (long long)plain);
            before = p;
            if (t < s.tiles) plain += s.blocks(c, t) + c.extra;
        }
        first.push_back(total);
        total += s.prefix(c, s.tiles) * n_kv;
    }
    EXPECT(total >= 0, "a list of cost %lld", (long long)total);
    if (total <= 0) return;
    std::map<std::tuple<int, int, int>, std::vector<int>> seen;         // (sequence, head, tile): how often each block
    const int64_t share = (total + ctas - 1) / ctas;
    for (int cta = 0; cta < ctas; ++cta) {
        Run r{};
        const int64_t lo = share * cta;
        r.share = share;
        r.left = total - lo < share ? total - lo : share;
        if (r.left <= 0) continue;
        for (r.b = B - 1; r.b > 0 && (first[r.b] > lo || load_seq(a, r.b, c).tiles == 0); --r.b) {}
        r.s = load_seq(a, r.b, c);
        const int64_t one = r.s.prefix(c, r.s.tiles);
        if (one <= 0) { EXPECT(false, "cost %lld belongs to no sequence", (long long)lo); continue; }
        r.h = (int)((lo - first[r.b]) / one);
        const int64_t in = (lo - first[r.b]) % one;
        while (r.tile + 1 < r.s.tiles && r.s.prefix(c, r.tile + 1) <= in) ++r.tile;
        r.skip = (int)(in - r.s.prefix(c, r.tile));
        Walk w(a, r, c);
        while (w.next()) {
            if (w.b >= B) { EXPECT(false, "CTA %d of %d walks past the last sequence", cta, ctas); break; }
            EXPECT(w.tokens() > 0 && w.j0 >= 0 && w.j0 < w.j1 && w.j1 <= w.blocks, "CTA %d: blocks %d .. %d of %d, %d tokens", cta, w.j0, w.j1, w.blocks, w.tokens());
            auto& blocks = seen[{w.b, w.h, w.tile - 1}];
            blocks.resize(w.blocks);
            for (int j = w.j0; j < w.j1; ++j) ++blocks[j];
        }
    }
    for (int b = 0; b < B; ++b) {
        const Seq s = load_seq(a, b, c);
        for (int h = 0; h < n_kv; ++h)
            for (int t = 0; t < s.tiles; ++t) {
                const auto& blocks = seen[{b, h, t}];
                EXPECT((int)blocks.size() == s.blocks(c, t), "sequence %d of %d (new %d, positions %d), head %d, tile %d: nobody's", b, B, n[b], lens[b], h, t);
                for (int times : blocks) EXPECT(times == 1, "sequence %d, head %d, tile %d: a block %d times", b, h, t, times);
            }
    }
}

static Cut tiles_cut(int group) { return Cut(128 / group * 2, TILE_KEYS_LOG, 2); }
static Cut few_cut(int group) { return Cut(FEW_TILE / group, FEW_KEYS_LOG, 1); }
static void both(const std::vector<int>& n, const std::vector<int>& L, int group, int n_kv, int ctas_tiles, int ctas_few) {
    for (int cuts = 0; cuts < 2; ++cuts) {
        walk_all(n, L, group, n_kv, tiles_cut(group), FEW_TILE, INT32_MAX, ctas_tiles, cuts);      // the two halves of one call
        walk_all(n, L, group, n_kv, few_cut(group), 0, FEW_TILE, ctas_few, cuts);
        walk_all(n, L, group, n_kv, tiles_cut(group), 0, INT32_MAX, ctas_tiles, cuts);             // all by one kernel
        walk_all(n, L, group, n_kv, few_cut(group), 0, INT32_MAX, ctas_few, cuts);
    }
}

int main() {
    // rows of a padded batch (one token, no position) beside a chunk, at each end and in the middle
    for (int at = 0; at < 12; ++at) {
        std::vector<int> n(12, 1), L(12, 0);
        n[at] = 512, L[at] = 1512;
        for (int i = 0; i < 12; i += 5) if (i != at) L[i] = 300;
        both(n, L, 4, 8, 80, 68);
    }
    both({1, 300, 1, 1}, {0, 700, 40, 90}, 4, 8, 100, 48);
    both({1, 1, 300, 1}, {40, 90, 100, 7}, 4, 8, 100, 48);              // a chunk of more tokens than positions
    both({300, 1, 1}, {0, 40, 90}, 4, 8, 100, 48);
    std::mt19937 gen(1);
    auto below = [&](int k) { return (int)(gen() % (unsigned)k); };
    const int groups[] = {1, 2, 3, 4, 6, 8, 9, 16};
    for (int round = 0; round < 1500; ++round) {
        const int B = 1 + below(30), group = groups[below(8)], n_kv = 1 + below(8);
        std::vector<int> n, L;
        for (int b = 0; b < B; ++b) {
            const int kind = below(4);
            n.push_back(kind == 0 ? 0 : kind == 1 ? 1 : kind == 2 ? 1 + below(20) : 1 + below(700));
            const int length = below(5);
            L.push_back(length == 0 ? 0 : length == 1 ? below(n[b] + 1) : n[b] + below(length == 2 ? 10 : 1500));
        }
        both(n, L, group, n_kv, 1 + below(148), 1 + below(148));
    }
    if (failures) printf("%d in all\n", failures);
    return failures != 0;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no CUDA compiler")
def test_runs_cover_the_list(tmp_path):
    src, exe = tmp_path / "list.cu", tmp_path / "list"
    src.write_text(SOURCE)
    subprocess.run([NVCC, "-O2", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{ROOT}/mixtral_offloading_b200/csrc", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
