"""Chunks beside single tokens in one call where a sequence has fewer positions than new tokens: the idle rows of a padded batch (one
token, no position) and chunks of more tokens than positions.  Rows that see nothing are 0, and every other row is what it is without
them, wherever such a sequence stands.  Bounds as in test_paged_attention.py."""
import itertools

import pytest
import torch

from mixtral_offloading_b200 import _cabi
from tests.test_paged_attention import DEV, Problem, check, reference

pytestmark = pytest.mark.gpu
FORMS = [(32, 8, 128, torch.bfloat16), (16, 1, 64, torch.float16), (9, 3, 128, torch.float16), (4, 4, 64, torch.bfloat16)]


def run(lens, new, H, n_kv, D, dtype, page=16):
    p = Problem(lens, new, H, n_kv, D, page, dtype, seed=len(lens))
    want, bound = p.want()
    spoiled = torch.full((96 << 20,), float("nan"), device=DEV)       # what the call's workspace is made of
    del spoiled
    out = torch.full_like(p.q, 7.25)
    p.paged(out=out)
    check(out, want, bound, (lens, new))
    for b, (L, n) in enumerate(zip(lens, new)):
        assert (out[p.cu[b]:p.cu[b] + max(0, n - L)] == 0).all(), b


@pytest.mark.parametrize("H,n_kv,D,dtype", FORMS)
@pytest.mark.parametrize("at", [0, 5, 11])
def test_idle_rows_beside_a_chunk(H, n_kv, D, dtype, at):
    new, lens = [1] * 12, [300 if i % 5 == 2 else 0 for i in range(12)]
    chunk = 700 * n_kv // H                                            # rows of a head: as many as the rule of both kernels takes beside 11 tokens
    new[at], lens[at] = chunk, chunk + 1000
    run(lens, new, H, n_kv, D, dtype)


@pytest.mark.parametrize("H,n_kv,D,dtype", FORMS)
@pytest.mark.parametrize("at", [0, 5, 11])
@pytest.mark.parametrize("positions", [0, 1, 100])
def test_a_chunk_of_more_tokens_than_positions_beside_single_tokens(H, n_kv, D, dtype, at, positions):
    new, lens = [1] * 12, [40 + 90 * i for i in range(12)]
    new[at], lens[at] = 150, positions
    run(lens, new, H, n_kv, D, dtype)


def test_a_padded_batch_beside_chunks():
    run([700] * 20 + [0] * 11 + [1512], [1] * 20 + [1] * 11 + [512], 32, 8, 128, torch.bfloat16)
    run([0, 700, 40, 90], [1, 300, 1, 1], 32, 8, 128, torch.bfloat16)
    run([0] * 15 + [400] + [0] * 16, [1] * 15 + [300] + [1] * 16, 32, 8, 128, torch.bfloat16)
    run([0] * 4, [1, 300, 1, 1], 32, 8, 128, torch.bfloat16)           # nobody sees anything


def test_a_captured_step_with_a_padded_batch():
    """Eight rows of a table, a chunk in front: requests come and go, rows without one have one token and no position."""
    p = Problem([900] + [500] * 7, [200] + [1] * 7, 32, 8, 128, 16, torch.bfloat16)
    out = torch.zeros_like(p.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.paged(out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.paged(out=out)
    for first, rest in ((900, [0] * 7), (200, [500, 0, 0, 3, 0, 1, 0]), (50, [0, 0, 0, 0, 0, 0, 500]), (0, [500] * 7), (0, [0] * 7), (900, [500] * 7)):
        lens = [first] + rest
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(2.5)
        g.replay()
        torch.cuda.synchronize()
        check(out, *reference(p.q, [k[:L] for k, L in zip(p.ks, lens)], [v[:L] for v, L in zip(p.vs, lens)], p.cu, 128 ** -0.5), lens)


def test_random_lengths():
    gen = torch.Generator().manual_seed(11)
    draw = lambda hi: int(torch.randint(0, hi + 1, (1,), generator=gen))
    for i in range(40):
        B = 2 + draw(30)
        new = [draw(3) if draw(4) else 30 + draw(250) for _ in range(B)]
        lens = [(0, draw(n), n + draw(9), n + draw(600))[draw(3)] for n in new]
        if sum(new):
            run(lens, new, *FORMS[i % len(FORMS)])


def test_no_wait_ran_out():
    assert _cabi.lib().hqm_device_error() == 0
