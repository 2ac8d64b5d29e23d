"""How the attention kernel of many rows hands blocks of keys and values from the warp that copies them to the two that issue the
products (csrc/attn_tiles.cu), step by step on the host in random orders: barriers that know their phase's parity only, copies and
products that end when they like.  Every product has to find its own block, and every step has to end.  With one ring for keys and
values, where each of the two warps waits for every second item only, products find older blocks: the model shows it."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

SOURCE = r"""
#include "attn.cuh"
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>
using namespace hqm::attn;

struct Barrier {
    int count = 1, pending = 1;
    uint32_t phase = 0;
    void arrive() { if (--pending == 0) { ++phase; pending = count; } }
    bool over(uint32_t parity) const { return (phase & 1) != parity; }         // what a wait for this parity finds
};
struct Later { int left; int kind, slot, item, tile; };                         // something that the hardware ends on its own

static std::mt19937 gen;
static int below(int n) { return (int)(gen() % (unsigned)n); }

// Items of keys and of values: their buffers and the parities of their waits.  SHARED: one ring of five, keys and values in turn.
template <bool SHARED>
struct Rings {
    static int buffer(bool v, uint32_t i) { return SHARED ? Ring<5>::buffer(2 * i + v) : v ? 3 + Ring<2>::buffer(i) : Ring<3>::buffer(i); }
    static uint32_t copied(bool v, uint32_t i) { return SHARED ? Ring<5>::copied(2 * i + v) : v ? Ring<2>::copied(i) : Ring<3>::copied(i); }
    static uint32_t used(bool v, uint32_t i) { return SHARED ? Ring<5>::used(2 * i + v) : v ? Ring<2>::used(i) : Ring<3>::used(i); }
    static bool wraps(bool v, uint32_t i) { return SHARED ? 2 * i + v >= 5 : i >= (v ? 2u : 3u); }
};

// 0: all well, 1: a product found another block, 2: nothing moves any more
template <bool SHARED>
static int simulate(int blocks, int tiles, int s_buffers, int slow) {
    typedef Rings<SHARED> R;
    Barrier full[5], empty[5], s_full[2], s_read[2], p_full[2], o_done[2];
    int holds[5] = {-1, -1, -1, -1, -1};                                         // 2 * block + (1 for values); -1 while a copy is on its way
    std::vector<Later> copies, s_queue, o_queue;                                 // (products of one warp end in their order)
    // where each warp is: the next thing it waits for
    uint32_t c_block = 0, c_v = 0, s_block = 0, s_tile = 0, o_block = 0, o_tile = 0;
    bool s_copied = false, o_copied = false;
    uint32_t made[2] = {0, 0}, w_block[2] = {0, 0}, w_step[2] = {0, 0};
    int idle = 0;
    auto done = [&] {
        for (int t = 0; t < tiles; ++t) if (w_block[t] < (uint32_t)blocks) return false;
        return o_block == (uint32_t)blocks && copies.empty() && s_queue.empty() && o_queue.empty();
    };
    while (!done()) {
        if (++idle > 100000) return 2;
        const int who = below(7);
        if (who == 0) {                                                          // the copies
            if (c_block == (uint32_t)blocks) continue;
            const int slot = R::buffer(c_v, c_block);
            if (R::wraps(c_v, c_block) && !empty[slot].over(R::used(c_v, c_block))) continue;
            holds[slot] = -1;
            copies.push_back({1 + (below(slow) ? below(4) : below(400)), 0, slot, (int)(2 * c_block + c_v), 0});
            if (c_v) ++c_block;
            c_v ^= 1;
        } else if (who == 1) {                                                   // S = Q K^T
            if (s_block == (uint32_t)blocks) continue;
            const int slot = R::buffer(false, s_block);
            if (!s_copied) { s_copied = full[slot].over(R::copied(false, s_block)); if (!s_copied) continue; }
            const int b = s_buffers == 2 ? s_tile : 0;
            if (made[b] > 0 && !s_read[b].over((made[b] + 1) & 1)) continue;
            ++made[b];
            if (holds[slot] != (int)(2 * s_block)) return 1;
            s_queue.push_back({1 + below(20), 1, slot, (int)s_block, (int)s_tile});
            if (++s_tile == (uint32_t)tiles) { s_tile = 0; ++s_block; s_copied = false; s_queue.push_back({1, 3, slot, 0, 0}); }
        } else if (who == 2) {                                                   // O += p V
            if (o_block == (uint32_t)blocks) continue;
            const int slot = R::buffer(true, o_block);
            if (!o_copied) { o_copied = full[slot].over(R::copied(true, o_block)); if (!o_copied) continue; }
            if (!p_full[o_tile].over(o_block & 1)) continue;
            if (holds[slot] != (int)(2 * o_block + 1)) return 1;
            o_queue.push_back({1 + below(20), 2, slot, (int)o_block, (int)o_tile});
            if (++o_tile == (uint32_t)tiles) { o_tile = 0; ++o_block; o_copied = false; o_queue.push_back({1, 3, slot, 0, 0}); }
        } else if (who <= 4) {                                                   // weights of a tile
            const int t = who - 3;
            if (t >= tiles || w_block[t] == (uint32_t)blocks) continue;
            if (w_step[t] == 0) {
                if (!s_full[t].over(w_block[t] & 1)) continue;
                s_read[s_buffers == 2 ? t : 0].arrive();
            } else {
                if (w_block[t] > 0 && !o_done[t].over((w_block[t] - 1) & 1)) continue;
                p_full[t].arrive();
                ++w_block[t];
            }
            w_step[t] ^= 1;
        } else if (who == 5) {                                                   // a copy of any age
            if (copies.empty()) continue;
            const int i = below((int)copies.size());
            if (--copies[i].left > 0) { idle = 0; continue; }
            holds[copies[i].slot] = copies[i].item;
            full[copies[i].slot].arrive();
            copies.erase(copies.begin() + i);
        } else {                                                                 // the oldest product of either warp
            auto& q = below(2) ? s_queue : o_queue;
            if (q.empty()) continue;
            if (--q[0].left > 0) { idle = 0; continue; }
            const Later e = q[0];
            q.erase(q.begin());
            if (e.kind == 1 && holds[e.slot] != 2 * e.item) return 1;            // until its end
            if (e.kind == 2 && holds[e.slot] != 2 * e.item + 1) return 1;
            if (e.kind == 1) s_full[e.tile].arrive();
            if (e.kind == 2) o_done[e.tile].arrive();
            if (e.kind == 3) empty[e.slot].arrive();
        }
        idle = 0;
    }
    return 0;
}

int main(int argc, char** argv) {
    const bool shared = argc > 1 && !strcmp(argv[1], "shared");
    int wrong[3] = {0, 0, 0};
    for (int seed = 0; seed < 4000; ++seed) {
        gen.seed(seed);
        const int blocks = 1 + below(40), tiles = 1 + below(2), s_buffers = 1 + below(2), slow = 2 + below(30);
        ++wrong[shared ? simulate<true>(blocks, tiles, s_buffers, slow) : simulate<false>(blocks, tiles, s_buffers, slow)];
    }
    printf("%d of 4000 orders go wrong, %d stop\n", wrong[1], wrong[2]);
    return wrong[1] + wrong[2] > 0;
}
"""


@pytest.mark.skipif(not os.path.exists(NVCC), reason="no CUDA compiler")
def test_every_product_finds_its_own_block(tmp_path):
    src, exe = tmp_path / "ring.cu", tmp_path / "ring"
    src.write_text(SOURCE)
    subprocess.run([NVCC, "-O2", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{ROOT}/mixtral_offloading_b200/csrc", "-o", str(exe), str(src)], check=True)
    run = lambda *args: subprocess.run([str(exe), *args], capture_output=True, text=True, timeout=300)
    out = run()
    assert out.returncode == 0, out.stdout
    assert run("shared").returncode == 1                            # (the model sees what it is there for)


def test_the_kernel_has_a_ring_for_each():
    text = open(os.path.join(ROOT, "mixtral_offloading_b200", "csrc", "attn_tiles.cu")).read()
    assert "K_RING = 3, V_RING = 2;" in text                       # what the model above has
    for role, ring, other in (("S = Q K^T ----", "KRing", "v_full"), ("O += p V ----", "VRing", "k_full")):
        body = text.split("// ---- " + role, 1)[1].split("// ----", 1)[0]
        assert f"{ring}::copied(at)" in body and f"{ring}::buffer(at)" in body and other not in body
