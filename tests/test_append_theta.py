"""Thetas that fp32 does not have (models stretched to longer contexts), at far positions: angles from all of theta's 64 bits."""
import math

import pytest
import torch

from mixtral_offloading_b200 import rope_append_paged
from tests.test_paged_tables import DEV, turned


@pytest.mark.gpu
@pytest.mark.parametrize("theta", [26914.93, 1e4 * 8 ** (128 / 126), 1e6 / 3, 1e6, 500000.0])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("fallback", [False, True])
def test_theta_in_64_bits(theta, dtype, D, fallback):
    gen = torch.Generator().manual_seed(7)
    T, H, n_kv, page = 64, 4, 2, 16
    rnd = lambda h: torch.randn(T, h, D, generator=gen).to(dtype).to(DEV)
    q, k, v = rnd(H), rnd(n_kv), rnd(n_kv)
    kp, vp = (torch.zeros(4, n_kv, page, D, dtype=dtype, device=DEV) for _ in range(2))
    positions = torch.randint(1 << 19, 1 << 20, (T,), generator=gen).to(torch.int32).to(DEV)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    p = torch.nn.Parameter(q, requires_grad=False) if fallback else q   # (of another class: the checks and the call from Python)
    out = rope_append_paged(p, k, v, kp, vp, positions, slots, theta)
    # as in test_paged_tables.py: one rounding; an angle's fraction, sine and cosine in fp32
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    for got, x in ((out, q), (kp.transpose(1, 2).reshape(T, n_kv, D), k)):
        want = turned(x, positions, theta)
        assert ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * x.double().abs().max() + tiny).all()


@pytest.mark.gpu
def test_thetas_that_cannot_be():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    pool = torch.zeros(2, 2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    i = torch.zeros(1, dtype=torch.int32, device=DEV)
    for theta in (0.0, -1e4, math.inf, math.nan, 1e39):
        with pytest.raises(ValueError):
            rope_append_paged(x, x, x, pool[0], pool[1], i, i, theta)
