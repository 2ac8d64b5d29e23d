"""Results that share memory with what is read: refused on the host, before anything is launched (the addresses here are none)."""
import ctypes as C
import os
import subprocess

import pytest

from mixtral_offloading_b200 import _cabi

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
    return 0;
}
"""


def test_pages_against_a_stretch(tmp_path):
    src, exe = tmp_path / "overlap.cpp", tmp_path / "overlap"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", f"-I{ROOT}/mixtral_offloading_b200/csrc", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
