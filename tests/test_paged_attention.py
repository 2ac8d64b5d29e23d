"""Attention of new tokens over pages and over packed prompts against its definition in 64 bits.

Bounds.  With weights w (softmax, 64 bits) a result is sum w v.  The kernels round a weight to the type before its product with
v and the result once more: half a step u = eps / 2 of |sum w v|, and of sum w |v|.  Scores are fp32 sums of head_dim products:
off by at most (head_dim + 2) 2^-24 of scale sum |q k|, which moves weight and total by that share each; exp2 and the sums of
weights add less than 2^-20."""
import itertools

import pytest
import torch

from mixtral_offloading_b200 import _cabi, paged_attention, prompt_attention

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def reference(q, ks, vs, cu, scale):
    """(sum w v, its bound) in 64 bits; ks[b], vs[b]: (L, n_kv, D) of sequence b, the new tokens last."""
    T, H, D = q.shape
    out, bound = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    u = torch.finfo(q.dtype).eps / 2
    for b, (k, v) in enumerate(zip(ks, vs)):
        lo, hi = cu[b], cu[b + 1]
        n, L = hi - lo, k.shape[0]
        if n == 0 or L == 0:
            continue
        group = H // k.shape[1]
        kk, vv = (t.double().repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))      # (H, L, D)
        qq = q[lo:hi].double().transpose(0, 1)
        seen = torch.arange(L, device=q.device)[None, :] <= L - n + torch.arange(n, device=q.device)[:, None]
        s = (qq @ kk.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
        w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        o, mag = w @ vv, w @ vv.abs()
        size = (qq.abs() @ kk.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        out[lo:hi] = o.transpose(0, 1)
        bound[lo:hi] = (u * o.abs() + (u * (1 + u) + 2 * (size * (D + 2) * 2.0 ** -24 + 2.0 ** -20)) * mag).transpose(0, 1)
    return out, bound + 1e-30 + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps


def check(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= bound).all(), f"{what}: {(off / bound).max().item():.3f} of the bound"


def pages_of(ks, page, gen, spare=3, poison=float("nan")):
    """A pool with the sequences' rows (L, n_kv, D) in pages of a random order, everything else `poison`; (pages, table)."""
    n_kv, D = ks[0].shape[1:]
    counts = [-(-k.shape[0] // page) for k in ks]
    pool = torch.full((sum(counts) + spare, n_kv, page, D), poison, dtype=ks[0].dtype, device=DEV)
    order = torch.randperm(pool.shape[0], generator=gen).tolist()
    table = torch.full((len(ks), max(counts + [1]) + 1), -7, dtype=torch.int32)
    for b, k in enumerate(ks):
        for i in range(counts[b]):
            p = order.pop()
            table[b, i] = p
            part = k[i * page:(i + 1) * page]
            pool[p, :, :part.shape[0]] = part.transpose(0, 1)
    return pool, table.to(DEV)


def refill(pool, table, ks, page):
    for b, k in enumerate(ks):
        for i in range(-(-k.shape[0] // page)):
            part = k[i * page:(i + 1) * page]
            pool[int(table[b, i]), :, :part.shape[0]] = part.transpose(0, 1)


class Problem:
    def __init__(self, lens, new, H, n_kv, D, page, dtype, seed=0, q_std=1.0):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(dtype).to(DEV)
        self.cu = list(itertools.accumulate(new, initial=0))
        self.q = rnd(self.cu[-1], H, D, std=q_std)
        self.ks, self.vs = [rnd(L, n_kv, D) for L in lens], [rnd(L, n_kv, D) for L in lens]
        self.page = page
        if page:
            self.k_pages, self.table = pages_of(self.ks, page, gen)
            self.v_pages = torch.full_like(self.k_pages, float("nan"))
            refill(self.v_pages, self.table, self.vs, page)
        self.cu_seqlens = torch.tensor(self.cu, dtype=torch.int32, device=DEV)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.max_new = max(new)

    def paged(self, **kw):
        return paged_attention(self.q, self.k_pages, self.v_pages, self.table, self.cu_seqlens, self.kv_lens,
                               kw.pop("max_new", self.max_new), **kw)

    def want(self, scale=None):
        return reference(self.q, self.ks, self.vs, self.cu, self.q.shape[-1] ** -0.5 if scale is None else scale)


HEADS = [(32, 8), (4, 4), (16, 2), (12, 2), (14, 2), (16, 1), (9, 3), (40, 1), (128, 1)]


@pytest.mark.parametrize("H,n_kv", HEADS)
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (128, torch.float16), (64, torch.float16)])
def test_single_tokens(H, n_kv, D, dtype):
    lens = [1, 2, 63, 64, 65, 128, 129, 500, 17, 1000]
    p = Problem(lens, [1] * len(lens), H, n_kv, D, 16, dtype)
    check(p.paged(), *p.want())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
def test_page_sizes(page):
    lens, new = [1, page - 1, page, page + 1, 3 * page + 5, 700], [1, 2, 1, 3, 2, 1]
    p = Problem(lens, new, 8, 2, 128, page, torch.bfloat16, seed=page)
    check(p.paged(), *p.want(), what="few")
    new = [min(n * 41, L) for n, L in zip(new, lens)]
    p = Problem(lens, new, 8, 2, 128, page, torch.bfloat16, seed=page + 1)
    check(p.paged(), *p.want(), what="chunks")


@pytest.mark.parametrize("H,n_kv", HEADS)
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_chunks(H, n_kv, D, dtype):
    lens = [1, 40, 128, 129, 257, 600, 300, 31, 513]
    new = [1, 40, 127, 5, 256, 17, 1, 31, 200]
    p = Problem(lens, new, H, n_kv, D, 32, dtype)
    check(p.paged(), *p.want())


@pytest.mark.parametrize("H,n_kv", HEADS)
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.bfloat16), (128, torch.float16), (64, torch.float16)])
def test_prompts(H, n_kv, D, dtype):
    new = [1, 2, 3, 17, 64, 127, 128, 129, 300, 1, 515]
    p = Problem(new, new, H, n_kv, D, 0, dtype)
    k, v = torch.cat(p.ks), torch.cat(p.vs)
    check(prompt_attention(p.q, k, v, p.cu_seqlens), *p.want())
    check(prompt_attention(p.q, k, v, p.cu_seqlens, max(new), scale=0.3), *p.want(0.3))


def test_one_token_prompts():
    new = [1] * 40
    p = Problem(new, new, 8, 2, 128, 0, torch.bfloat16)
    got = prompt_attention(p.q, torch.cat(p.ks), torch.cat(p.vs), p.cu_seqlens, 1)
    assert torch.equal(got, torch.cat(p.vs).repeat_interleave(4, 1))         # one position: its value


def test_a_neighbour_that_is_not_finite():
    """Packed prompts: the tile of one prompt reaches into the next one."""
    new = [5, 130, 7, 70]
    p = Problem(new, new, 8, 2, 128, 0, torch.bfloat16)
    want, bound = p.want()
    k, v = torch.cat(p.ks), torch.cat(p.vs)
    for b in (0, 2):
        for value in (float("nan"), float("inf"), -float("inf")):
            kk, vv = k.clone(), v.clone()
            kk[p.cu[b]:p.cu[b + 1]], vv[p.cu[b]:p.cu[b + 1]] = value, value
            got = prompt_attention(p.q, kk, vv, p.cu_seqlens)
            for c in (1, 3):
                rows = slice(p.cu[c], p.cu[c + 1])
                check(got[rows], want[rows], bound[rows], f"{b} {value}")


@pytest.mark.parametrize("chunk", [1, 3, 90])
def test_rows_that_see_nothing_are_zero_and_rows_behind_the_last_sequence_stay(chunk):
    """Sequences without tokens, without positions, and with fewer positions than new tokens."""
    lens, new = [0, 200, 3, 0, 77, 1], [chunk, 0, chunk, 0, chunk, chunk]
    p = Problem(lens, new, 8, 2, 128, 16, torch.bfloat16)
    want, bound = p.want()
    T = p.cu[-1]
    q = torch.cat([p.q, torch.full((9, 8, 128), float("nan"), dtype=p.q.dtype, device=DEV)])
    out = torch.full((T + 9, 8, 128), 7.25, dtype=p.q.dtype, device=DEV)
    got = paged_attention(q, p.k_pages, p.v_pages, p.table, p.cu_seqlens, p.kv_lens, chunk, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[T:] == 7.25).all()
    check(out[:T], want, bound)
    for b, (L, n) in enumerate(zip(lens, new)):
        blind = out[p.cu[b]:p.cu[b] + max(0, n - L)]
        assert (blind == 0).all()


def test_nothing_to_do():
    p = Problem([3], [1], 4, 2, 64, 16, torch.bfloat16)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert paged_attention(p.q[:0], p.k_pages, p.v_pages, p.table, p.cu_seqlens * 0, p.kv_lens, 1).shape == (0, 4, 64)
    out = torch.full_like(p.q, 3.0)
    paged_attention(p.q, p.k_pages, p.v_pages, p.table, p.cu_seqlens * 0, p.kv_lens, 1, out=out)      # no sequence has tokens
    paged_attention(p.q, p.k_pages, p.v_pages, p.table[:0], one, none, 1, out=out)                    # no sequences
    prompt_attention(p.q, p.q[:, :2], p.q[:, :2], one, out=out)
    assert (out == 3).all()


def test_strides():
    """Views of one projection's output, heads in front of tokens, pages of both kinds in one pool."""
    new, lens = [70, 3, 20], [70, 90, 21]
    H, n_kv, D = 8, 2, 128
    p = Problem(lens, new, H, n_kv, D, 16, torch.bfloat16)
    T = p.cu[-1]
    fused = torch.randn(T, H + 2 * n_kv + 1, D, device=DEV).to(torch.bfloat16)
    fused[:, :H] = p.q
    both = torch.stack([p.k_pages, p.v_pages], 1)                      # (pages, 2, ...)
    wide = torch.full((3, 50), -1, dtype=torch.int32, device=DEV)
    wide[:, :p.table.shape[1]] = p.table
    got = paged_attention(fused[:, :H], both[:, 0], both[:, 1], wide[:, :p.table.shape[1]], p.cu_seqlens, p.kv_lens, 70)
    check(got, *p.want())
    assert torch.equal(got, p.paged())
    ks = [fused[a:b, H:H + n_kv] for a, b in zip(p.cu, p.cu[1:])]
    vs = [fused[a:b, H + n_kv:H + 2 * n_kv] for a, b in zip(p.cu, p.cu[1:])]
    q2 = p.q.transpose(0, 1).contiguous().transpose(0, 1)              # heads in front of tokens
    got = prompt_attention(q2, fused[:, H:H + n_kv], fused[:, H + n_kv:H + 2 * n_kv], p.cu_seqlens, 70)
    check(got, *reference(p.q, ks, vs, p.cu, D ** -0.5))


def test_large_scores_and_a_peaked_softmax():
    """Maxima that grow and fall along the keys by hundreds: the running maximum has to follow."""
    lens, new = [900, 700], [150, 1]
    for order in (1, -1):
        p = Problem(lens, new, 8, 2, 128, 64, torch.bfloat16, q_std=8.0)
        for b, k in enumerate(p.ks):
            ramp = torch.linspace(0.1, 6.0, k.shape[0], device=DEV)
            if order < 0:
                ramp = ramp.flip(0)
            p.ks[b] = (k * ramp[:, None, None]).to(torch.bfloat16)
        refill(p.k_pages, p.table, p.ks, 64)
        check(p.paged(), *p.want(), what=str(order))


@pytest.mark.parametrize("new", [1, 3, 90])
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_a_key_that_is_not_finite_reaches_the_rows_that_see_it(new, D, dtype):
    """Every column of a block of keys in turn; rows that do not see it, and the other sequence, are as without it."""
    L, group = 200, 4
    for value in (float("nan"), float("inf"), -float("inf")):
        for at in list(range(L - new - 1 if new > 1 else 100, L, 7)) + [L - 1, 0]:
            p = Problem([L, 150], [new, new], 8, 2, D, 16, dtype, seed=at)
            want, bound = p.want()
            p.ks[0][at, :, 5] = value
            refill(p.k_pages, p.table, p.ks, 16)
            got = p.paged()
            score = p.q[:new, :, 5].double() * value                   # NaN, or infinite with the sign of q
            sees = torch.arange(new, device=DEV)[:, None] + L - new >= at
            lost = sees & ~(score == -float("inf"))
            assert torch.isnan(got[:new][lost]).all(), (value, at)
            clean = torch.cat([~sees.expand(new, 8), torch.ones(new, 8, dtype=torch.bool, device=DEV)])
            check(got[clean], want[clean], bound[clean], (value, at))
            assert torch.isfinite(got[:new][~lost]).all()


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_the_largest_values_in_masked_places(D, dtype):
    """Weights of masked places are exactly 0: values as large as the type has, in a later position, leave a row as it is."""
    for new in (4, 90):
        p = Problem([300, 40], [new, 2], 8, 2, D, 16, dtype)
        want, bound = p.want()
        p.vs[0][-1] = torch.finfo(dtype).max
        p.ks[0][-1] = torch.finfo(dtype).max * 2.0 ** -12              # (finite scores)
        refill(p.v_pages, p.table, p.vs, 16)
        refill(p.k_pages, p.table, p.ks, 16)
        got = p.paged()
        rows = list(range(new - 1)) + [new, new + 1]
        check(got[rows], want[rows], bound[rows], new)


@pytest.mark.parametrize("pages", [1, 3, 5, 6, 40])
@pytest.mark.parametrize("H,n_kv,D", [(32, 8, 128), (9, 3, 64), (4, 4, 128)])
def test_tables_of_few_pages(pages, H, n_kv, D):
    """Rows of the table from one block on: units that are not cut, and the same ones cut where the table is wide."""
    page = 64
    lens = [pages * page, pages * page - 5, 1]
    for new in (1, 40):
        p = Problem(lens, [min(new, L) for L in lens], H, n_kv, D, page, torch.bfloat16, seed=pages)
        p.table = p.table[:, :pages].contiguous()
        check(p.paged(), *p.want(), what=(pages, new))
        wide = torch.cat([p.table, p.table.new_full((3, 50), -1)], 1)
        check(paged_attention(p.q, p.k_pages, p.v_pages, wide, p.cu_seqlens, p.kv_lens, p.max_new), *p.want(), what="wide")


def test_a_row_of_equal_scores():
    """q = 0: the mean of what a row sees, whatever the keys are; -3e38 as the keys' lowest values does not matter."""
    p = Problem([333, 140], [60, 1], 8, 2, 128, 16, torch.bfloat16)
    p.q.zero_()
    check(p.paged(), *p.want())


def test_entries_outside_the_pool_read_as_zeros():
    p = Problem([100, 60], [3, 1], 8, 2, 128, 16, torch.bfloat16)
    want, bound = p.want()
    for bad in (-1, p.k_pages.shape[0], 2 ** 31 - 1):
        table = p.table.clone()
        table[1, 1] = bad
        got = paged_attention(p.q, p.k_pages, p.v_pages, table, p.cu_seqlens, p.kv_lens, 3)
        check(got[:3], want[:3], bound[:3])
        ks, vs = [t.clone() for t in p.ks], [t.clone() for t in p.vs]
        ks[1][16:32], vs[1][16:32] = 0, 0
        check(got, *reference(p.q, ks, vs, p.cu, 128 ** -0.5))


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 elements, its last pages in use."""
    n_kv, page, D = 8, 256, 128
    pages = (1 << 32) // (n_kv * page * D) + 40
    pool = torch.empty(pages, n_kv, page, D, dtype=torch.bfloat16, device=DEV)
    for new in (1, 50):
        p = Problem([700, 300], [new, new], 32, n_kv, D, page, torch.bfloat16)
        table = p.table.clone()
        for b, n in enumerate((3, 2)):
            for i in range(n):
                far = pages - 1 - (3 * b + i)
                pool[far] = p.k_pages[int(p.table[b, i])]
                table[b, i] = far
        got = paged_attention(p.q, pool, pool, table, p.cu_seqlens, p.kv_lens, new)
        check(got, *reference(p.q, p.ks, p.ks, p.cu, D ** -0.5))


def test_a_long_cache_is_split_and_joined_with_the_same_bits_each_time():
    p = Problem([40000], [1], 32, 8, 128, 64, torch.bfloat16)
    first = p.paged()
    check(first, *p.want())
    for _ in range(5):
        assert torch.equal(p.paged(), first)
    p = Problem([9000, 5, 7000], [3, 2, 300], 32, 8, 128, 64, torch.bfloat16)
    first = p.paged()
    check(first, *p.want())
    for _ in range(5):
        assert torch.equal(p.paged(), first)


def test_many_sequences():
    gen = torch.Generator().manual_seed(5)
    lens = torch.randint(1, 60, (700,), generator=gen).tolist()
    new = [min(L, int(n)) for L, n in zip(lens, torch.randint(0, 4, (700,), generator=gen))]
    p = Problem(lens, new, 8, 2, 64, 16, torch.float16)
    check(p.paged(), *p.want())


@pytest.mark.parametrize("B", [31, 32, 33, 64, 65, 100, 1100])
def test_numbers_of_sequences(B):
    """Around the 32 that a warp looks at at once; empty sequences, single tokens, a few and many rows."""
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 200, (B,), generator=gen).tolist()
    for most in (1, 30):
        new = [min(L, int(n)) for L, n in zip(lens, torch.randint(0, most + 1, (B,), generator=gen))]
        p = Problem(lens, new, 8, 2, 64, 16, torch.bfloat16, seed=B)
        check(p.paged(), *p.want(), what=(B, most))
    one = [0] * (B - 1) + [150]                                            # all of it in the last sequence
    p = Problem([max(L, 1) for L in lens[:-1]] + [190], one, 8, 2, 64, 16, torch.bfloat16, seed=B)
    check(p.paged(), *p.want(), what="last")


@pytest.mark.parametrize("H,n_kv,D,dtype", [(32, 8, 128, torch.bfloat16), (16, 1, 64, torch.float16), (12, 2, 128, torch.float16)])
def test_single_tokens_beside_chunks(H, n_kv, D, dtype):
    """Sequences of up to 16 rows per key/value head and longer ones in one call, around that line, empty ones among them."""
    group = H // n_kv
    line = 16 // group
    new = [1] * 20 + [300, 0, line, line + 1, 1, 64, 0, 2, 1] + [1] * 12
    lens = [n + (37 * i) % 700 for i, n in enumerate(new)]
    p = Problem(lens, new, H, n_kv, D, 16, dtype)
    check(p.paged(), *p.want())


def test_one_kind_of_sequences_alone_and_a_captured_call_of_both():
    """A call made for both kinds of sequences that has only one of them, by its lengths or in a replay."""
    p = Problem([700, 9, 40], [300, 5, 5], 32, 8, 128, 16, torch.bfloat16)                # all of many rows
    check(p.paged(), *p.want(), what="many")
    p = Problem([700, 300, 40, 90], [200, 1, 2, 1], 32, 8, 128, 16, torch.bfloat16)
    out = torch.zeros_like(p.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.paged(out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.paged(out=out)
    for new in ([200, 1, 2, 1], [0, 1, 2, 1], [200, 0, 0, 0], [100, 100, 0, 4], [0, 0, 0, 0], [1, 200, 1, 1]):
        lens = [max(n, L) for n, L in zip(new, (700, 300, 40, 90))]
        lens = [min(L, k.shape[0]) for L, k in zip(lens, p.ks)]
        cu = list(itertools.accumulate(new, initial=0))
        p.cu_seqlens.copy_(torch.tensor(cu, dtype=torch.int32))
        p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(2.5)
        g.replay()
        torch.cuda.synchronize()
        want, bound = reference(p.q, [k[:L] for k, L in zip(p.ks, lens)], [v[:L] for v, L in zip(p.vs, lens)], cu, 128 ** -0.5)
        check(out[:cu[-1]], want[:cu[-1]], bound[:cu[-1]], new)
        assert (out[cu[-1]:] == 2.5).all()


def test_max_new_is_a_bound_only():
    p = Problem([300, 40, 7], [3, 1, 2], 32, 8, 128, 16, torch.bfloat16)
    want, bound = p.want()
    for max_new in (3, 4, 5, 30, 1000):
        check(p.paged(max_new=max_new), want, bound, str(max_new))


def test_a_captured_call_follows_the_lengths():
    """Lengths change between replays; two graphs of different sizes replayed at once on two streams."""
    graphs = []
    for new, seed in ((1, 1), (40, 2)):
        p = Problem([600, 900, 50], [new] * 3, 32, 8, 128, 16, torch.bfloat16, seed=seed)
        out = torch.zeros_like(p.q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            p.paged(out=out)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.paged(out=out)
        graphs.append((p, out, g, new))
    for lens in ([600, 900, 50], [599, 64, 41], [40, 300, 50]):
        for p, out, g, new in graphs:
            p.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(3):
            for (p, out, g, new), s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for p, out, g, new in graphs:
            ks, vs = [k[:L] for k, L in zip(p.ks, lens)], [v[:L] for v, L in zip(p.vs, lens)]
            check(out, *reference(p.q, ks, vs, p.cu, 128 ** -0.5), what=str((lens, new)))


def test_two_streams_at_once():
    ps = [Problem([3000 + 100 * i, 700], [n, n], 32, 8, 128, 64, torch.bfloat16, seed=i) for i, n in enumerate((1, 60))]
    wants = [p.want() for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                outs.append(p.paged())
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        check(out, *wants[i % 2])


def test_no_wait_ran_out():
    assert _cabi.lib().hqm_device_error() == 0
