"""Results and inputs that begin on a 16-byte boundary which is no 32-byte one: what the header allows.  The bits are those of tensors
that begin where an allocation does, and nothing beside a result is touched."""
import pytest
import torch

from mixtral_offloading_b200 import _cabi, paged_attention, prompt_attention
from tests.test_paged_attention import DEV, Problem, check

pytestmark = pytest.mark.gpu


def shifted(t, by=8):
    """A contiguous copy of t that begins `by` elements into its storage."""
    room = torch.zeros(t.numel() + 2 * by, dtype=t.dtype, device=t.device)
    room[by:by + t.numel()] = t.reshape(-1)
    out = room[by:by + t.numel()].view(t.shape)
    assert out.data_ptr() % 32 == 16
    return out


class Result:
    def __init__(self, like, by=8):
        self.room = torch.full((like.numel() + 2 * by,), 3.5, dtype=like.dtype, device=like.device)
        self.by, self.out = by, self.room[by:by + like.numel()].view(like.shape)
        assert self.out.data_ptr() % 32 == 16

    def untouched(self):
        return bool((self.room[:self.by] == 3.5).all() and (self.room[-self.by:] == 3.5).all())


@pytest.mark.parametrize("H,n_kv,D,dtype", [(32, 8, 128, torch.bfloat16), (16, 16, 64, torch.float16), (9, 3, 128, torch.float16), (16, 1, 64, torch.bfloat16)])
@pytest.mark.parametrize("lens,new", [([400, 90, 17], [1, 1, 1]), ([400, 290, 17], [300, 130, 17]), ([5000, 900], [200, 300]),
                                      ([900] + [60 * i for i in range(1, 12)], [250] + [1] * 11)],
                         ids=["few", "many", "cut", "both"])
def test_over_pages(H, n_kv, D, dtype, lens, new):
    p = Problem(lens, new, H, n_kv, D, 16, dtype)
    want = p.paged()
    r = Result(p.q)
    p.paged(out=r.out)
    assert torch.equal(r.out, want) and r.untouched()
    check(r.out, *p.want())
    r = Result(p.q)
    paged_attention(shifted(p.q), shifted(p.k_pages), shifted(p.v_pages), p.table, p.cu_seqlens, p.kv_lens, p.max_new, out=r.out)
    assert torch.equal(r.out, want) and r.untouched()


@pytest.mark.parametrize("H,n_kv,D,dtype", [(32, 8, 128, torch.bfloat16), (16, 16, 64, torch.float16), (9, 3, 128, torch.float16)])
@pytest.mark.parametrize("new", [[3, 1], [17], [300, 5, 129], [3000]], ids=str)
def test_over_prompts(H, n_kv, D, dtype, new):
    p = Problem(new, new, H, n_kv, D, 0, dtype)
    k, v = torch.cat(p.ks), torch.cat(p.vs)
    want = prompt_attention(p.q, k, v, p.cu_seqlens, max(new))
    for q2, k2, v2 in ((p.q, k, v), (shifted(p.q), shifted(k), shifted(v))):
        r = Result(p.q)
        prompt_attention(q2, k2, v2, p.cu_seqlens, max(new), out=r.out)
        assert torch.equal(r.out, want) and r.untouched()
    check(want, *p.want())


def test_no_wait_ran_out():
    assert _cabi.lib().hqm_device_error() == 0
