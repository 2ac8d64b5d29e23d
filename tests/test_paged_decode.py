"""PagedDecode against MixtralDecodeModel, which feeds one sequence at a time over a cache of its own.

Two experts, both of which every token takes: no choice of experts can turn a rounding into another token's path.  Each side is
held to 2e-2 of the largest logit against the oracle after two layers (tests/test_decoder_layer_oracle.py), so they are within
4e-2 of one another."""
import pytest
import torch

from mixtral_offloading_b200 import DecoderLayerDecode, MixtralDecodeModel, PagedDecode, ResidentMoe, _cabi
from tests.helpers import random_layer
from tests.test_decode_attention import _Cfg, build
from tests.test_gpu_parity import make_expert

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
VOCAB, MAX_LEN, TOL = 300, 160, 4e-2


@pytest.fixture(scope="module")
def model():
    n_heads, n_kv, hidden, ffn, E, L = 4, 2, 512, 1792, 2, 2
    g = torch.Generator().manual_seed(3)
    lns = [(1 + 0.1 * torch.randn(hidden, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(L + 1)]
    layers = []
    for l in range(L):
        attn, _, _ = build(n_heads, n_kv, MAX_LEN, seed=40 + 7 * l)
        experts = [make_expert(hidden, ffn, tuple(random_layer(n, k, 2, 16, 900 + 30 * l + 3 * e + i) for i, (n, k) in
                                                  enumerate(((ffn, hidden), (hidden, ffn), (ffn, hidden))))) for e in range(E)]
        gate = torch.nn.Linear(hidden, E, bias=False, dtype=torch.bfloat16, device=DEV)
        gate.weight.data.copy_((0.1 * torch.randn(E, hidden, generator=g)).to(torch.bfloat16))
        layers.append(DecoderLayerDecode(attn, ResidentMoe(_Cfg(hidden, ffn, E), l, gate, experts), lns[l + 1]))
    embed = torch.randn(VOCAB, hidden, generator=g).to(torch.bfloat16).to(DEV)
    head = (0.05 * torch.randn(VOCAB, hidden, generator=g)).to(torch.bfloat16).to(DEV)
    return MixtralDecodeModel(embed, layers, lns[0], head)


def tokens(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def close(row, model, fed):
    want = model.prefill(fed)[0].float()
    return float((row.float() - want).abs().max() / want.abs().max()) < TOL


@pytest.mark.parametrize("page_size", [16, 64])
def test_steps_of_prompts_chunks_and_single_tokens(model, page_size):
    p = PagedDecode(model, 4, 512 // page_size, page_size, MAX_LEN)
    fed = [[], [], [], []]
    steps = [(5, 70, 0, 1), (1, 1, 33, 1), (0, 20, 1, 1), (60, 1, 1, 1), (1, 1, 0, 7)]
    for i, new in enumerate(steps):
        feed = [tokens(n, 100 * i + b) for b, n in enumerate(new)]
        logits = p.step(feed)
        fed = [f + n for f, n in zip(fed, feed)]
        assert p.kv_lens.tolist() == p.lens == [len(f) for f in fed]
        active = [b for b, n in enumerate(new) if n]
        assert logits.shape == (len(active), VOCAB)
        for row, b in zip(logits, active):
            assert close(row, model, fed[b]), (i, b)
    # rejected tokens and a request that has ended; its pages serve another one
    p.truncate([30, 0, len(fed[2]), len(fed[3])])
    fed = [fed[0][:30], [], fed[2], fed[3]]
    feed = [tokens(2, 1), tokens(90, 2), [], tokens(1, 3)]
    logits = p.step(feed)
    fed = [f + n for f, n in zip(fed, feed)]
    for row, b in zip(logits, (0, 1, 3)):
        assert close(row, model, fed[b]), b
    held = sum(-(-len(f) // page_size) for f in fed)
    assert p.free_count.item() == p.pages - held
    pages = [x for b, f in enumerate(fed) for x in p.block_table[b, :-(-len(f) // page_size)].tolist()]
    assert sorted(pages + p.free_pages[:p.pages - held].tolist()) == list(range(p.pages))
    assert _cabi.lib().hqm_device_error() == 0


def test_generate_serves_requests_of_different_lengths(model):
    p = PagedDecode(model, 5, 40, 16, MAX_LEN)
    prompts = [tokens(n, 50 + n) for n in (3, 60, 17)]
    out = p.generate(prompts, 6, chunk=25)
    assert [len(o) for o in out] == [6, 6, 6]
    for prompt, o in zip(prompts, out):                            # every token is (nearly) the best one behind what was fed
        for i, t in enumerate(o):
            want = model.prefill(prompt + o[:i])[0].float()
            assert want.max() - want[t] <= 2 * TOL * want.abs().max()
    assert p.lens == [0] * 5 and p.free_count.item() == 40
    assert p.generate(prompts, 6, chunk=25) == out
    short = p.generate(prompts, 6, chunk=25, eos_token_id=out[1][2])
    assert short[1] == out[1][:out[1].index(out[1][2]) + 1] and p.free_count.item() == 40


def test_what_does_not_fit_is_refused(model):
    p = PagedDecode(model, 2, 4, 16, 50)
    for bad in ([[1]], [[], []], [[1] * 51, []], [[1] * 40, [1] * 20], ):
        with pytest.raises(ValueError):
            p.step(bad)
    p.step([[1] * 40, [2] * 16])
    with pytest.raises(ValueError):
        p.step([[1] * 9, [1]])
    for bad in ([41, 0], [0], [-1, 0]):
        with pytest.raises(ValueError):
            p.truncate(bad)
    for bad in ([], [[1], []], [[1]] * 3):
        with pytest.raises(ValueError):
            p.generate(bad, 3)
    assert p.lens == [40, 16] == p.kv_lens.tolist()


def test_shapes_and_tokens_that_cannot_be_are_refused(model):
    for bad in ((0, 4, 16, 50), (2, 0, 16, 50), (2, 4, 8, 50), (2, 4, 48, 50), (2, 4, 16, 0)):
        with pytest.raises(ValueError):
            PagedDecode(model, *bad)
    p = PagedDecode(model, 2, 4, 16, 50)
    for bad in (-1, VOCAB):
        with pytest.raises(ValueError):
            p.step([[1, bad], []])
    assert p.lens == [0, 0] == p.kv_lens.tolist() and p.free_count.item() == 4


def test_a_pool_that_runs_out_is_empty_again(model):
    p = PagedDecode(model, 2, 4, 16, 50)
    with pytest.raises(ValueError):
        p.generate([tokens(30, 1), tokens(31, 2)], 8)
    assert p.lens == [0, 0] == p.kv_lens.tolist() and p.free_count.item() == 4
    assert [len(o) for o in p.generate([tokens(3, 1), tokens(5, 2)], 4)] == [4, 4]
