"""Results that share memory with what is read: refused on the host, before anything is launched (the addresses here are none)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from mixtral_offloading_b200 import _cabi, rope_append_paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MB = 1 << 20
PAGE = 2 * 16 * 128                          # elements of a page


def attention(**change):
    ok = dict(out=1 * MB, q=2 * MB, k=16 * MB, v=32 * MB, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128, k_page=PAGE,
              v_page=PAGE, block_table=4096, table_stride=4, cu_seqlens=4096, kv_lens=4096, tokens=3, sequences=1, max_new=3, n_heads=4,
              n_kv_heads=2, head_dim=128, pages=9, page_size=16, max_pages=4, dtype=0, scale=0.1)
    return _cabi.lib().hqm_paged_attention(C.byref(_cabi.HqmAttention(**dict(ok, **change))), C.c_void_p(4096), 0, None)


def refused(rc):
    return rc == _cabi.HQM_ERR_ARG and "shares memory" in _cabi.last_error()


def test_attention_into_its_own_pages():
    size = 3 * 512 * 2                                                 # bytes of out
    for pool in (16 * MB, 32 * MB):
        pages = 2 * 9 * PAGE
        for out in (pool, pool + 2 * PAGE, pool + pages - 16, pool - size + 16):
            assert refused(attention(out=out)), out
        for out in (pool + pages, pool - size):                       # beside it: refused for another reason (scratch, or no device)
            assert not refused(attention(out=out)), out
    # pages that lie apart: what is between them is not theirs
    far = dict(k_page=16 * PAGE, v_page=16 * PAGE, v=16 * MB + 2 * PAGE)
    for page in (0, 3, 8):
        at = 16 * MB + 2 * 16 * PAGE * page
        for out in (at, at + 2 * PAGE + 16, at + 2 * 2 * PAGE - 16, at - size + 16):
            assert refused(attention(out=out, **far)), (page, out)
        assert not refused(attention(out=at + 2 * 2 * PAGE, **far)) and not refused(attention(out=at + 2 * 16 * PAGE - size, **far))


def append(**change):
    ok = dict(q_out=1 * MB, k_out=0, q=2 * MB, k=3 * MB, v=4 * MB, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128,
              k_pages=16 * MB, v_pages=32 * MB, k_page=PAGE, v_page=PAGE, positions=4096, slots=4096, tokens=3, n_heads=4, n_kv_heads=2, head_dim=128,
              pages=9, page_size=16, dtype=0, rope_theta=1e4)
    return _cabi.lib().hqm_rope_append_paged(C.byref(_cabi.HqmPagedAppend(**dict(ok, **change))), None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would be launched on addresses that are none")
def test_append_refuses_what_its_threads_would_race_for():
    q_size, k_size, pool = 3 * 512 * 2, 3 * 256 * 2, 2 * 9 * PAGE
    fused = dict(q=2 * MB, k=2 * MB + 1024, v=2 * MB + 1536, q_token=1024, k_token=1024, v_token=1024)       # one projection's output
    for change in (dict(q_out=2 * MB + 16), dict(q_out=2 * MB + q_size - 16), dict(q_out=2 * MB - q_size + 16),        # q, shifted
                   dict(q_out=2 * MB, q_token=1024), dict(q_out=2 * MB, q_head=256), dict(fused, q_out=2 * MB),           # q, laid out otherwise
                   dict(q_out=3 * MB), dict(q_out=4 * MB + k_size - 16), dict(q_out=16 * MB), dict(q_out=32 * MB + pool - 16),
                   dict(k_out=2 * MB), dict(k_out=4 * MB), dict(k_out=1 * MB + q_size - 16), dict(k_out=3 * MB + 16), dict(k_out=3 * MB, k_token=512),
                   dict(k_out=16 * MB + 64), dict(k_out=32 * MB - k_size + 16), dict(fused, k_out=2 * MB + 1024),
                   dict(q=16 * MB), dict(k=16 * MB + pool - 16), dict(v=32 * MB), dict(v_pages=16 * MB), dict(v_pages=16 * MB + pool - 16),
                   dict(k_page=4 * PAGE, v_page=4 * PAGE, v_pages=16 * MB + 2 * 8 * PAGE), dict(k_page=4 * PAGE, v_page=2 * PAGE, v_pages=16 * MB + 2 * PAGE)):
        assert append(**change) == _cabi.HQM_ERR_ARG and "shares memory" in _cabi.last_error(), change


@pytest.mark.gpu
def test_append_in_place_and_from_one_projection():
    """What stays allowed, with one pool for keys and values, against separate tensors."""
    dev = torch.device("cuda:0")
    gen = torch.Generator().manual_seed(4)
    T, H, n_kv, D, page = 37, 8, 2, 128, 16
    fused = torch.randn(T, H + 2 * n_kv, D, generator=gen).to(torch.bfloat16).to(dev)
    positions = torch.arange(T, dtype=torch.int32, device=dev)
    q, k, v = fused[:, :H], fused[:, H:H + n_kv], fused[:, H + n_kv:]
    kp, vp = (torch.zeros(5, n_kv, page, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    want, want_k = torch.empty_like(q.contiguous()), torch.empty_like(k.contiguous())
    rope_append_paged(q, k, v, kp, vp, positions, positions + 8, 1e4, out=want, k_out=want_k)
    both = torch.zeros(5, 2, n_kv, page, D, dtype=torch.bfloat16, device=dev)
    q2, k2 = q.contiguous(), k.contiguous()
    rope_append_paged(q2, k2, v, both[:, 0], both[:, 1], positions, positions + 8, 1e4, out=q2, k_out=k2)
    assert torch.equal(q2, want) and torch.equal(k2, want_k) and torch.equal(both[:, 0], kp) and torch.equal(both[:, 1], vp)
    row = fused[:1].clone()                                            # one token: all of it is contiguous
    q1, k1 = row[:, :H], row[:, H:H + n_kv]
    rope_append_paged(q1, k1, row[:, H + n_kv:], kp, vp, positions[:1], positions[:1] + 8, 1e4, out=q1, k_out=k1)
    assert torch.equal(q1, want[:1]) and torch.equal(k1, want_k[:1])
    for bad in (lambda: rope_append_paged(q2, k2, k2, kp, vp, positions, positions, 1e4, k_out=k2),
                lambda: rope_append_paged(q, k, v, kp, vp, positions, positions, 1e4, out=fused.view(-1)[:T * H * D].view(T, H, D)),
                lambda: rope_append_paged(q, k, v, kp, kp, positions, positions, 1e4)):
        with pytest.raises(ValueError):
            bad()


SOURCE = r"""
#include "overlap.h"
#include <cstdio>
#include <vector>
using namespace hqm;
static void* at(int64_t element) { return reinterpret_cast<void*>((uintptr_t)(4096 + 2 * element)); }
int main() {
    // every stretch of up to 9 elements against pages of up to 4, element by element
    for (int elements = 1; elements <= 4; ++elements)
        for (int stride = elements; stride <= 7; ++stride)
            for (int count = 1; count <= 4; ++count) {
                std::vector<bool> theirs(80);
                for (int i = 0; i < count; ++i) for (int e = 0; e < elements; ++e) theirs[20 + i * stride + e] = true;
                for (int from = 0; from < 60; ++from)
                    for (int n = 1; n <= 9; ++n) {
                        bool want = false;
                        for (int e = from; e < from + n; ++e) want = want || theirs[e];
                        if (Pages{at(20), count, stride, elements}.meets(elements_at(at(from), n)) != want)
                            return printf("%d pages of %d, %d apart, against %d elements from %d\n", count, elements, stride, n, from - 20), 1;
                    }
            }
    // pages against pages: any strides, in front of and behind one another
    for (int n1 = 1; n1 <= 3; ++n1) for (int s1 = n1; s1 <= 6; ++s1) for (int c1 = 1; c1 <= 4; ++c1)
        for (int n2 = 1; n2 <= 3; ++n2) for (int s2 = n2; s2 <= 6; ++s2) for (int c2 = 1; c2 <= 4; ++c2)
            for (int from = 0; from < 70; ++from) {
                std::vector<int> theirs(120);
                bool want = false;
                for (int i = 0; i < c1; ++i) for (int e = 0; e < n1; ++e) theirs[30 + i * s1 + e] = 1;
                for (int i = 0; i < c2; ++i) for (int e = 0; e < n2; ++e) want = want || theirs[from + i * s2 + e];
                const Pages one{at(30), c1, s1, n1}, two{at(from), c2, s2, n2};
                if (c1 > 1 && c2 > 1 && s1 != s2) {                    // the stretches decide
                    want = elements_at(one.at, (c1 - 1) * s1 + n1).meets(elements_at(two.at, (c2 - 1) * s2 + n2));
                }
                if (one.meets(two) != want || two.meets(one) != want)
                    return printf("%d pages of %d, %d apart, and %d of %d, %d apart, from %d\n", c1, n1, s1, c2, n2, s2, from - 30), 1;
            }
    // rows of any strides, also backwards
    for (int token = -12; token <= 12; ++token)
        for (int head = -6; head <= 6; ++head) {
            const Stretch s = rows_at(at(60), 3, 2, token, head, 2);
            int64_t lo = 1000, hi = -1000;
            for (int t = 0; t < 3; ++t) for (int h = 0; h < 2; ++h) for (int e = 0; e < 2; ++e) {
                const int64_t x = 60 + t * token + h * head + e;
                lo = x < lo ? x : lo, hi = x > hi ? x : hi;
            }
            if (s.from != elements_at(at(lo), 1).from || s.to != elements_at(at(hi), 1).to) return printf("rows %d, %d\n", token, head), 1;
        }
    return 0;
}
"""


def test_pages_against_a_stretch(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/mixtral_offloading_b200/csrc", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
