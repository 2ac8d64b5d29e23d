"""Rows whose largest weight stands above very many small ones: each of them is below the steps that fp16 has beside 1, together they are
not.

Bounds: those of test_paged_attention.py (half a step u of the result and of every weight, scores in fp32), and for weights below the
type's normal numbers half of its last step, N 2^-25 2^-7 max |v| of N keys where the largest weight is held as 2^7 or more."""
import math

import pytest
import torch

from mixtral_offloading_b200 import _cabi, prompt_attention
from tests.test_paged_attention import DEV, Problem, check, reference, refill

pytestmark = pytest.mark.gpu
N, PAGE = 131072, 1024


def problem(lens, new, D, dtype, below, peak, at=8.0):
    """One key/value head, two query heads: key `peak` scores 1 = the largest, every other one 2^-below of it; values of 1 there, -1 + noise elsewhere."""
    p = Problem(lens, new, 2, 1, D, PAGE, dtype, seed=3)
    gen = torch.Generator().manual_seed(5)
    step = below * math.log(2) * math.sqrt(D) / at                     # q k / sqrt(D) is that much lower in e's powers
    p.q = torch.zeros_like(p.q)
    p.q[..., 0] = at
    for b, L in enumerate(lens):
        k = torch.zeros_like(p.ks[b])
        k[:, 0, 0] = 1.0 - step
        k[peak % L, 0, 0] = 1.0
        v = (-1 + 0.25 * torch.randn(L, 1, D, generator=gen)).to(dtype).to(DEV)
        v[peak % L] = 1.0
        p.ks[b], p.vs[b] = k, v
    refill(p.k_pages, p.table, p.ks, PAGE)
    refill(p.v_pages, p.table, p.vs, PAGE)
    return p


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("below", [20.0, 25.2])
@pytest.mark.parametrize("peak", [0, 70000])
@pytest.mark.parametrize("lens,new", [([N], [1]), ([N], [30]), ([N, 90, 400], [30, 1, 1])], ids=["few", "many", "both"])
def test_one_peak_above_a_flat_rest(lens, new, peak, below, dtype):
    for D in (64, 128):
        p = problem(lens, new, D, dtype, below, peak)
        want, bound = p.want()
        small = max(lens) * 2.0 ** -32 * 2.5 if dtype == torch.float16 else 0.0
        check(p.paged(), want, bound + small, (D, below))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_one_peak_at_the_beginning_of_a_long_prompt(D, dtype):
    """Units that one CTA works on from the first key to the last, so that all of a row's weights refer to the peak's."""
    p = problem([N], [1], D, dtype, 25.2, 0)
    q = p.q[:1].expand(N, 2, D).contiguous()
    got = prompt_attention(q, p.ks[0], p.vs[0], torch.tensor([0, N], dtype=torch.int32, device=DEV))
    for end in (N, N // 2 + 77, 5000):
        want, bound = reference(q[:64], [p.ks[0][:end]], [p.vs[0][:end]], [0, 64], D ** -0.5)
        check(got[end - 64:end], want, bound + (end * 2.0 ** -32 * 2.5 if dtype == torch.float16 else 0.0), end)


@pytest.mark.parametrize("new", [1, 30])
def test_maxima_far_from_nothing(new):
    """fp16 scores up to 2^23: one key far above the others, then all of them alike."""
    for size, k_top in ((64.0, 64.0), (512.0, 1024.0), (2048.0, 2048.0), (2048.0, 4096.0)):
        p = problem([700], [new], 128, torch.float16, 1.0, 5)
        p.q[..., 0] = size
        k = torch.full_like(p.ks[0], 0)
        k[:, 0, 0] = k_top / 2
        k[5, 0, 0] = k_top                                             # size k_top / 2 / sqrt(128): 180 of e's powers above the rest at the least
        p.ks = [k]
        refill(p.k_pages, p.table, p.ks, PAGE)
        for scale in (128 ** -0.5, 1.0):                               # half a step of the one weight, half a step of the result 1
            assert ((p.paged(scale=scale).double() - 1).abs() <= 2 * 2.0 ** -11).all(), (size, scale)
        k[:, 0, 0] = k_top                                             # all alike: their mean
        refill(p.k_pages, p.table, p.ks, PAGE)
        seen = 700 - new + 1 + torch.arange(new, device=DEV)
        want = (torch.cumsum(p.vs[0][:, 0].double(), 0)[seen - 1] / seen[:, None])[:, None].expand(new, 2, 128)
        # half a step of the result and of the weights, which are all the same; 700 additions of fp32 for the sum and for the total
        mag = (torch.cumsum(p.vs[0][:, 0].double().abs(), 0)[seen - 1] / seen[:, None])[:, None]
        for scale in (128 ** -0.5, 1.0):
            assert ((p.paged(scale=scale).double() - want).abs() <= 2.0 ** -11 * (want.abs() + mag) + 2 * 700 * 2.0 ** -24 * mag).all(), (size, scale)


def test_no_wait_ran_out():
    assert _cabi.lib().hqm_device_error() == 0
