"""Block tables, slot maps and the append into pages against plain Python, and what the operators refuse."""
import ctypes as C
import math

import pytest
import torch

from mixtral_offloading_b200 import (_cabi, paged_attention, paged_reserve, paged_truncate, prompt_attention,
                                     rope_append_paged)

DEV = torch.device("cuda:0")
gpu = pytest.mark.gpu


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Model:
    """The cache in plain Python."""

    def __init__(self, B, pages, page, max_pages, order):
        self.page, self.max_pages, self.free = page, max_pages, list(order)
        self.table, self.lens = [[-1] * max_pages for _ in range(B)], [0] * B
        self.pages = pages

    def reserve(self, new, tokens):
        need = [-(-(l + n) // self.page) - -(-l // self.page) for l, n in zip(self.lens, new)]
        B = len(new)
        none = ([0] * (B + 1), self.lens[:], [-1] * tokens, [-1] * tokens)
        if any(n < 0 or l + n > self.max_pages * self.page for l, n in zip(self.lens, new)):
            return none + (-1,)
        if sum(new) > tokens:
            return none + (-2,)
        if sum(need) > len(self.free):
            return none + (sum(need) - len(self.free),)
        cu, positions, slots = [0], [], []
        for b, n in enumerate(new):
            held = -(-self.lens[b] // self.page)
            for i in range(need[b]):
                self.table[b][held + i] = self.free.pop()
            for i in range(self.lens[b], self.lens[b] + n):
                positions.append(i)
                slots.append(self.table[b][i // self.page] * self.page + i % self.page)
            self.lens[b] += n
            cu.append(cu[-1] + n)
        pad = [-1] * (tokens - len(positions))
        return cu, self.lens[:], positions + pad, slots + pad, 0

    def truncate(self, keep):
        if any(k < 0 or k > l for k, l in zip(keep, self.lens)):
            return -1
        back = []
        for b, k in enumerate(keep):
            back += self.table[b][-(-k // self.page):-(-self.lens[b] // self.page)]
            self.lens[b] = k
        self.free += back[::-1]
        return 0


@gpu
@pytest.mark.parametrize("B,page,pages,most", [(1, 16, 40, 30), (5, 16, 60, 40), (64, 32, 900, 50), (700, 16, 9000, 30), (3, 7, 50, 20),
                                              (40, 64, 2000, 900), (3, 16, 2600, 8000)])
def test_tables_follow_a_plain_model(B, page, pages, most):
    gen = torch.Generator().manual_seed(B)
    order = torch.randperm(pages, generator=gen).tolist()
    max_pages = max(8, 4 * most // page)
    m = Model(B, pages, page, max_pages, order)
    table = torch.full((B, max_pages + 3), -1, dtype=torch.int32, device=DEV)[:, :max_pages]        # rows further apart than long
    lens, free, count = ints([0] * B), ints(order), ints([pages])
    seen = set()
    for step in range(40):
        rand = lambda hi: torch.randint(0, hi + 1, (B,), generator=gen).tolist()
        if step % 3 == 2:
            keep = [min(k, l) if step % 2 else k for k, l in zip(rand(4 * most), m.lens)]
            status = paged_truncate(table, lens, free, count, ints(keep), page)
            want = m.truncate(keep)
            assert status.item() == want
        else:
            new = rand(most if step % 2 else 2)
            if step == 7:
                new[B // 2] = -1
            tokens = sum(new) + (13 if step % 4 == 0 else 0) if step != 9 else max(0, sum(new) - 1)
            tokens = max(tokens, 0)
            got = paged_reserve(table, lens, free, count, ints(new), page, tokens)
            want = m.reserve(new, tokens)
            assert got.status.item() == want[4]
            for g, w in zip(got[:4], want):
                assert g.tolist() == w
            want = want[4]
        seen.add((want > 0) - (want < 0))
        assert lens.tolist() == m.lens and count.item() == len(m.free)
        assert free[:len(m.free)].tolist() == m.free
        held = [-(-l // page) for l in m.lens]
        for row, mine, n in zip(table.tolist(), m.table, held):
            assert row[:n] == mine[:n]
    assert 0 in seen


@gpu
def test_a_step_that_is_taken_back_leaves_the_stack_as_it_was():
    free = ints(list(range(100, 0, -1)))
    table, lens, count = ints([[0] * 20] * 3), ints([0, 0, 0]), ints([100])
    paged_reserve(table, lens, free, count, ints([33, 1, 70]), 16, 104)
    before = [t.clone() for t in (table, lens, free, count)]
    paged_reserve(table, lens, free, count, ints([16, 15, 200]), 16, 231)
    assert paged_truncate(table, lens, free, count, before[1], 16).item() == 0
    assert torch.equal(lens, before[1]) and torch.equal(count, before[3]) and torch.equal(free, before[2])


@gpu
def test_a_stack_that_cannot_be_right_is_refused():
    table, lens, free = ints([[0, 1, 2, 3]]), ints([20]), ints(list(range(8)))
    for count in (-1, 9):
        n = ints([count])
        got = paged_reserve(table, lens, free, n, ints([1]), 16, 1)
        assert got.status.item() == -3 and got.slots.tolist() == [-1] and n.item() == count
        assert paged_truncate(table, lens, free, n, ints([0]), 16).item() == -3
    n = ints([7])                                                   # two pages back on a stack with room for one
    assert paged_truncate(table, lens, free, n, ints([0]), 16).item() == -3
    assert lens.tolist() == [20] and free.tolist() == list(range(8))


@gpu
def test_no_sequences_and_no_tokens():
    none = ints([])
    table, free, count = torch.zeros(0, 4, dtype=torch.int32, device=DEV), ints([1, 2]), ints([2])
    got = paged_reserve(table, none, free, count, none, 16, 3)
    assert got.cu_seqlens.tolist() == [0] and got.slots.tolist() == [-1] * 3 and got.status.item() == 0
    assert paged_truncate(table, none, free, count, none, 16).item() == 0
    got = paged_reserve(table, none, free, count, none, 16, 5000)
    assert got.cu_seqlens.tolist() == [0] and got.slots.tolist() == [-1] * 5000 and got.positions.tolist() == [-1] * 5000
    got = paged_reserve(ints([[5, 0]]), ints([3]), free, count, ints([0]), 16, 0)
    assert got.cu_seqlens.tolist() == [0, 0] and got.positions.numel() == 0 and count.item() == 2


# ---- the append --------------------------------------------------------------------------------------------------------
def turned(x, positions, theta):
    """Rotate-half in 64 bits."""
    D = x.shape[-1]
    freq = torch.tensor([theta ** (-2 * d / D) for d in range(D // 2)], dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None, None] * freq
    a, b = x[..., :D // 2].double(), x[..., D // 2:].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,n_kv,D,page", [(1, 32, 8, 128, 16), (7, 4, 4, 64, 64), (300, 12, 2, 128, 32), (33, 16, 1, 64, 256)])
def test_rope_append(dtype, T, H, n_kv, D, page):
    gen = torch.Generator().manual_seed(T)
    pages = -(-2 * T // page) + 2
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(DEV)
    fused = rnd(T, H + 2 * n_kv, D)
    q, k, v = fused[:, :H], fused[:, H:H + n_kv], fused[:, H + n_kv:]
    kp, vp = rnd(pages, n_kv, page, D), rnd(pages, n_kv, page, D)
    positions = torch.randint(0, 1 << 20, (T,), generator=gen).to(torch.int32)
    positions[0] = 0
    slots = torch.randperm(pages * page, generator=gen)[:T].to(torch.int32)
    drop = torch.rand(T, generator=gen) < 0.2
    drop[0] = False
    slots[drop], positions[drop] = -1, -1
    positions, slots, drop = positions.to(DEV), slots.to(DEV), drop.to(DEV)
    want_k, want_v = kp.double(), vp.double()
    at = slots[~drop].long()
    want_k[at // page, :, at % page] = turned(k[~drop], positions[~drop], 1e6)
    want_v[at // page, :, at % page] = v[~drop].double()
    out = torch.full((T, H, D), 5.0, dtype=dtype, device=DEV)
    assert rope_append_paged(q, k, v, kp, vp, positions, slots, 1e6, out=out).data_ptr() == out.data_ptr()
    # one rounding; an angle's fraction, sine and cosine in fp32: 2^-21 of both products, and of what is as far below the type's steps
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    close = lambda got, want, mag: ((got.double() - want).abs() <= u * want.abs() + 2.0 ** -20 * mag + tiny).all()
    mag = fused.double().abs().max()
    assert close(out[~drop], turned(q[~drop], positions[~drop], 1e6), mag)
    assert (out[drop] == 5).all()
    assert close(kp, want_k, mag) and torch.equal(vp.double(), want_v)
    again = q.contiguous()
    assert torch.equal(rope_append_paged(again, k, v, kp, vp, positions, slots, 1e6, out=again)[~drop], out[~drop])     # in place
    k_out = torch.full((T, n_kv, D), 6.0, dtype=dtype, device=DEV)
    assert torch.equal(rope_append_paged(q, k, v, kp, vp, positions, slots, 1e6, k_out=k_out)[~drop], out[~drop])
    assert torch.equal(k_out[~drop], kp[at // page, :, at % page]) and (k_out[drop] == 6).all()
    again = k.contiguous()
    rope_append_paged(q, again, v, kp, vp, positions, slots, 1e6, k_out=again)
    assert torch.equal(again[~drop], k_out[~drop])


@gpu
def test_a_slot_beyond_the_pool_is_left_out():
    q, k = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=DEV), torch.ones(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    kp = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    vp = kp.clone()
    assert _cabi.lib().hqm_device_error() == 0
    rope_append_paged(q, k, k, kp, vp, ints([0, 0]), ints([32, 3]), 1e4)
    assert _cabi.lib().hqm_device_error() == 2 and _cabi.lib().hqm_device_error() == 0
    assert vp.sum().item() == 2 * 64 and (vp[0, :, 3] == 1).all()


@gpu
def test_tables_append_and_attention_as_a_step_uses_them():
    """Three sequences, prompts and single tokens, a rejected continuation: what the pages hold gives what plain lists give."""
    B, H, n_kv, D, page, theta = 3, 8, 2, 128, 16, 1e4
    gen = torch.Generator().manual_seed(3)
    kp = torch.full((40, n_kv, page, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    vp = kp.clone()
    table, lens, free, count = ints([[0] * 12] * B), ints([0] * B), ints(torch.randperm(40, generator=gen).tolist()), ints([40])
    ks, vs = [torch.zeros(0, n_kv, D, device=DEV) for _ in range(B)], [torch.zeros(0, n_kv, D, device=DEV) for _ in range(B)]
    for new, keep in (([50, 3, 0], None), ([1, 20, 0], None), ([1, 1, 33], None), ([5, 5, 5], [52, 29, 34]), ([1, 1, 1], None), ([0, 40, 2], None)):
        T = sum(new)
        q, k, v = (torch.randn(T, h, D, generator=gen).to(torch.bfloat16).to(DEV) for h in (H, n_kv, n_kv))
        step = paged_reserve(table, lens, free, count, ints(new), page, T)
        rq = rope_append_paged(q, k, v, kp, vp, step.positions, step.slots, theta)
        got = paged_attention(rq, kp, vp, table, step.cu_seqlens, step.kv_lens, max(new))
        assert step.status.item() == 0
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            rows = slice(at, at + n)
            pos = torch.arange(ks[b].shape[0], ks[b].shape[0] + n, device=DEV)
            assert step.positions[rows].tolist() == pos.tolist()
            ks[b] = torch.cat([ks[b], turned(k[rows], pos, theta).to(torch.bfloat16).float()])
            vs[b] = torch.cat([vs[b], v[rows].float()])
            kk, vv = (t.double().repeat_interleave(H // n_kv, 1).transpose(0, 1) for t in (ks[b], vs[b]))
            s = turned(q[rows], pos, theta).to(torch.bfloat16).double().transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(D)
            s = s.masked_fill(torch.arange(kk.shape[1], device=DEV)[None, :] > pos[:, None], float("-inf"))
            w = torch.softmax(s, -1)
            # half a step of the result, of every weight, of every rotated q and k (their scores: 2 * 2^-8 of sum |q k| / sqrt(D) at the most
            # where the two roundings fall apart by one step, which few do; a tenth of that bounds what is left of it in the weights)
            want, mag = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
            assert ((got[rows].double() - want).abs() <= 2.0 ** -8 * (want.abs() + mag) + 0.02 * mag + 1e-6).all()
            at += n
        if keep:
            assert paged_truncate(table, lens, free, count, ints(keep), page).item() == 0
            ks, vs = [t[:n] for t, n in zip(ks, keep)], [t[:n] for t, n in zip(vs, keep)]


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_the_library_refuses_what_it_cannot_do():
    """On the host, before anything is launched."""
    lib = _cabi.lib()
    some = C.c_void_p(4096)
    ok = dict(out=4096, q=4096, k=4096, v=4096, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128, k_page=4096,
              v_page=4096, block_table=4096, table_stride=4, cu_seqlens=4096, kv_lens=4096, tokens=3, sequences=1, max_new=3, n_heads=4,
              n_kv_heads=2, head_dim=128, pages=9, page_size=16, max_pages=4, dtype=0, scale=0.1)
    for change, word in ((dict(head_dim=96), "head_dim"), (dict(dtype=2), "dtype"), (dict(n_heads=5), "query heads"), (dict(n_kv_heads=0), "query heads"),
                         (dict(page_size=24), "power of two"), (dict(page_size=8), "power of two"), (dict(k_page=4095), "pages"),
                         (dict(table_stride=3), "pages"), (dict(max_pages=0), "pages"), (dict(pages=1 << 28), "pages"),
                         (dict(max_pages=1 << 28, table_stride=1 << 28), "pages"), (dict(q=0), "null"), (dict(kv_lens=0), "null"),
                         (dict(q_token=513), "16-byte"), (dict(k_page=4100), "16-byte"), (dict(v=4104), "16-byte"), (dict(tokens=-1), "tokens"),
                         (dict(tokens=1 << 31), "tokens"), (dict(max_new=-1), "at most"), (dict(scale=float("nan")), "scale"),
                         (dict(scale=0.0), "positive"), (dict(n_heads=258), "query heads")):
        call = _cabi.HqmAttention(**dict(ok, **change))
        assert lib.hqm_paged_attention(C.byref(call), some, 1 << 40, None) == _cabi.HQM_ERR_ARG, change
        assert word in _cabi.last_error(), (change, _cabi.last_error())
    for change in (dict(k_head=0), dict(v_token=-256)):
        call = _cabi.HqmAttention(**dict(ok, **change))
        assert lib.hqm_prompt_attention(C.byref(call), some, 1 << 40, None) == _cabi.HQM_ERR_ARG, change
    assert lib.hqm_prompt_attention(None, some, 1 << 40, None) == _cabi.HQM_ERR_ARG
    for change in (dict(tokens=0), dict(sequences=0), dict(max_new=0)):                         # nothing to do
        assert lib.hqm_paged_attention(C.byref(_cabi.HqmAttention(**dict(ok, **change))), None, 0, None) == 0
    ok = dict(q_out=4096, k_out=0, q=4096, k=4096, v=4096, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128, k_pages=4096,
              v_pages=4096, k_page=4096, v_page=4096, positions=4096, slots=4096, tokens=3, n_heads=4, n_kv_heads=2, head_dim=128, pages=9,
              page_size=16, dtype=0, rope_theta=1e4, reserved=0)
    for change in (dict(head_dim=80), dict(dtype=3), dict(page_size=12), dict(k_page=100), dict(rope_theta=0.0), dict(slots=0), dict(k_head=4),
                   dict(q=4098), dict(k_out=4100), dict(tokens=-1), dict(n_kv_heads=0)):
        call = _cabi.HqmPagedAppend(**dict(ok, **change))
        assert lib.hqm_rope_append_paged(C.byref(call), None) == _cabi.HQM_ERR_ARG, change
    assert lib.hqm_rope_append_paged(C.byref(_cabi.HqmPagedAppend(**dict(ok, tokens=0))), None) == 0
    reserve = lambda *tail: lib.hqm_paged_reserve(some, 8, some, some, some, some, some, some, some, some, some, *tail, None)
    for tail in ((16385, 8, 16, 100, 5), (-1, 8, 16, 100, 5), (4, 9, 16, 100, 5), (4, 0, 16, 100, 5), (4, 8, 0, 100, 5), (4, 8, 16, 0, 5),
                 (4, 8, 16, 1 << 28, 5), (4, 8, 16, 100, -1)):
        assert reserve(*tail) == _cabi.HQM_ERR_ARG, tail
    assert lib.hqm_paged_truncate(some, 8, some, some, None, some, some, 4, 8, 16, 100, None) == _cabi.HQM_ERR_ARG


def test_a_result_that_shares_memory_with_what_is_read_is_refused():
    lib = _cabi.lib()
    ok = dict(q=1 << 20, k=2 << 20, v=3 << 20, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256, v_head=128, k_page=4096, v_page=4096,
              block_table=4096, table_stride=4, cu_seqlens=4096, kv_lens=4096, tokens=3, sequences=1, max_new=3, n_heads=4, n_kv_heads=2,
              head_dim=128, pages=9, page_size=16, max_pages=4, dtype=0, scale=0.1)
    size = 3 * 512 * 2
    for out in (1 << 20, (1 << 20) + size - 16, (1 << 20) - size + 16):
        for entry in (lib.hqm_paged_attention, lib.hqm_prompt_attention):
            assert entry(C.byref(_cabi.HqmAttention(**dict(ok, out=out))), C.c_void_p(4096), 0, None) == _cabi.HQM_ERR_ARG
            assert "shares memory" in _cabi.last_error()
    for out in (2 << 20, (3 << 20) + 256):
        assert lib.hqm_prompt_attention(C.byref(_cabi.HqmAttention(**dict(ok, out=out))), C.c_void_p(4096), 0, None) == _cabi.HQM_ERR_ARG
        assert "shares memory" in _cabi.last_error()
    # right behind q: refused for another reason (no scratch, or no device), not for its place
    lib.hqm_paged_attention(C.byref(_cabi.HqmAttention(**dict(ok, out=(1 << 20) + size))), C.c_void_p(4096), 0, None)
    assert "shares memory" not in _cabi.last_error()


def test_no_cpu_path():
    t = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    pool = torch.zeros(2, 4, 16, 64, dtype=torch.bfloat16)
    for call in (lambda: prompt_attention(t, t, t, i), lambda: paged_attention(t, pool, pool, i[None], torch.zeros(2, dtype=torch.int32), i, 1),
                 lambda: rope_append_paged(t, t, t, pool, pool, i, i, 1e4), lambda: paged_reserve(i[None], i, i, i, i, 16, 1),
                 lambda: paged_truncate(i[None], i, i, i, i, 16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@gpu
def test_the_python_layer_refuses():
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    pool = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    cu, lens, table = ints([0, 3]), ints([5]), ints([[0, 1]])
    bad = [
        lambda: paged_attention(q.float(), pool, pool, table, cu, lens, 3),
        lambda: paged_attention(q, pool.half(), pool, table, cu, lens, 3),
        lambda: paged_attention(q[0], pool, pool, table, cu, lens, 3),
        lambda: paged_attention(q, pool.transpose(1, 2), pool.transpose(1, 2), table, cu, lens, 3),
        lambda: paged_attention(q, pool, pool[:3], table, cu, lens, 3),
        lambda: paged_attention(q, pool, pool, table.long(), cu, lens, 3),
        lambda: paged_attention(q, pool, pool, table, cu[:1], lens, 3),
        lambda: paged_attention(q, pool, pool, table.cpu(), cu, lens, 3),
        lambda: paged_attention(q, pool, pool, table, cu, lens, 3, out=q[:2]),
        lambda: paged_attention(q[..., ::2], pool[..., ::2], pool[..., ::2], table, cu, lens, 3),
        lambda: prompt_attention(q, k[:2], k[:2], cu),
        lambda: prompt_attention(q, k, k, cu.long()),
        lambda: prompt_attention(q[:, :3], k, k, cu),
        lambda: rope_append_paged(q, k, k, pool, pool, cu, cu, 1e4),
        lambda: rope_append_paged(q, k[:, :1], k[:, :1], pool, pool, ints([0, 1, 2]), ints([0, 1, 2]), 1e4),
        lambda: rope_append_paged(q, k, k, pool, pool, ints([0, 1, 2]), ints([0, 1, 2]), 1e4, k_out=q),
        lambda: paged_reserve(table, lens, ints([2, 3]), ints([2]), ints([1, 1]), 16, 2),
        lambda: paged_reserve(table, lens, ints([2, 3]), ints([2]), ints([1]), 16, -1),
        lambda: paged_truncate(table, lens, ints([2, 3]), ints([2, 0]), ints([1]), 16),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
