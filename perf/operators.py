"""The operators of the paged key/value cache as cases that can be timed: block tables and slot maps from request lengths,
rotary embedding with the append into pages, attention of new tokens over the pages, attention over whole packed prompts.

Heads are the ones the package is built around (32 query and 8 key/value heads of 128), and other generic layouts.  Lengths are
ragged: they come from the case (`lens` seeds them), the values and the order of the pages from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA = 1e6


def listed():
    heads = {"heads": 32, "kv_heads": 8, "dim": 128}
    return [
        # the tables of a decoding step of 64 requests
        {"name": "tables-decode-64", "kind": "tables", "sequences": 64, "context": 4000, "new": 1, "page": 16, "lens": 1},
        # the tables of 256 prompts that arrive together
        {"name": "tables-prompts-256", "kind": "tables", "sequences": 256, "context": 0, "new": 700, "page": 32, "lens": 2},
        # keys and values of a decoding step of 64 requests
        {"name": "append-decode-64", "kind": "append", "sequences": 64, "context": 8000, "new": 1, "page": 16, "dtype": "bf16", "lens": 3,
         **heads},
        # keys and values of 16 chunks far into their sequences
        {"name": "append-chunks-16", "kind": "append", "sequences": 16, "context": 100000, "new": 1024, "page": 64, "dtype": "bf16", "lens": 4,
         **heads},
        # one request, one token: the smallest call
        {"name": "paged-token-1x500", "kind": "paged", "sequences": 1, "context": 500, "new": 1, "page": 64, "dtype": "bf16", "lens": 5, **heads},
        # a decoding step of 64 requests of different lengths
        {"name": "paged-token-64", "kind": "paged", "sequences": 64, "context": 8192, "new": 1, "page": 64, "dtype": "bf16", "lens": 6, **heads},
        # one token behind a long document
        {"name": "paged-token-long", "kind": "paged", "sequences": 1, "context": 130001, "new": 1, "page": 16, "dtype": "fp16", "lens": 7, **heads},
        # chunks of prompts behind what is cached already
        {"name": "paged-chunks-8", "kind": "paged", "sequences": 8, "context": 4000, "new": 256, "page": 32, "dtype": "bf16", "lens": 8, **heads},
        # a serving step: two long chunks among 30 requests that decode
        {"name": "paged-mixed-32", "kind": "paged", "sequences": 32, "context": 4000, "new": 512, "chunks": 2, "page": 64, "dtype": "bf16",
         "lens": 9, **heads},
        # a short question
        {"name": "prompt-17", "kind": "prompt", "sequences": 1, "new": 17, "dtype": "bf16", "lens": 10, **heads},
        # 24 prompts in one pass, a head layout without sharing
        {"name": "prompt-packed-24", "kind": "prompt", "sequences": 24, "new": 1500, "dtype": "fp16", "lens": 11, "heads": 16, "kv_heads": 16,
         "dim": 64},
        # a long document
        {"name": "prompt-16001", "kind": "prompt", "sequences": 1, "new": 16001, "dtype": "bf16", "lens": 12, **heads},
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(("tables", "append", "paged", "paged", "paged", "prompt", "prompt"))
    case = {"kind": kind, "lens": rng.randint(1, 1 << 30)}
    if kind == "tables":
        new = _log_int(rng, 1, 700)
        return dict(case, sequences=_log_int(rng, 1, 256), context=rng.choice((0, _log_int(rng, 1, 8000))), new=new,
                    page=rng.choice((16, 32, 64, 128)))
    groups, kv = rng.choice(((4, 8), (4, 8), (1, 16), (8, 2), (6, 4), (16, 1)))
    case.update(heads=groups * kv, kv_heads=kv, dim=rng.choice((64, 128, 128)), dtype=rng.choice(("bf16", "bf16", "fp16")))
    if kind == "prompt":
        sequences = _log_int(rng, 1, 32)
        return dict(case, sequences=sequences, new=_log_int(rng, 1, int(12000 / math.sqrt(sequences))))
    case["page"] = rng.choice((16, 32, 64, 128, 256))
    if kind == "append":
        return dict(case, sequences=_log_int(rng, 1, 64), context=_log_int(rng, 1, 16000), new=_log_int(rng, 1, 256))
    form = rng.choice(("token", "token", "chunk", "mixed"))
    if form == "token":                                              # one token, or the few of a speculated continuation
        sequences = _log_int(rng, 1, 96)
        return dict(case, sequences=sequences, context=_log_int(rng, 1, min(130000, 524288 // sequences)), new=_log_int(rng, 1, 5))
    sequences = _log_int(rng, 2, 32)
    case.update(sequences=sequences, context=_log_int(rng, 1, 48000 // sequences), new=_log_int(rng, 6, min(2048, 6144 // sequences)))
    return dict(case, chunks=rng.randint(1, sequences)) if form == "mixed" else case


def _lengths(case):
    """(cached, new) tokens of every sequence.  One sequence, or one new token: as the case says; else between an eighth and all of it.
    With `chunks`, that many sequences have a chunk and the others one token."""
    rng = random.Random(case["lens"])
    n = case["sequences"]
    cached, new = [], []
    for b in range(n):
        most = case.get("context", 0)
        cached.append(most if n == 1 else rng.randint(most // 8, most))
        most = case["new"]
        if "chunks" in case and b % max(1, n // case["chunks"]) != 0:
            most = 1
        new.append(most if n == 1 or most < 6 else rng.randint(max(1, most // 8), most))
    return cached, new


def _ceil(a, b):
    return -(-a // b)


def _normal(gen, *shape, dtype):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=dtype)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cumulative(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    cached, new = _lengths(case)
    cu = _cumulative(new)
    s = {"case": case, "cached": cached, "new": new, "cu": cu, "cu_seqlens": _int(cu), "tokens": cu[-1], "max_new": max(new)}
    if case["kind"] == "prompt":
        dtype = DTYPES[case["dtype"]]
        s["q"] = _normal(gen, s["tokens"], case["heads"], case["dim"], dtype=dtype)
        s["k"], s["v"] = (_normal(gen, s["tokens"], case["kv_heads"], case["dim"], dtype=dtype) for _ in range(2))
        return s
    page = case["page"]
    # the pool: what the sequences hold, what they are about to, and a fifth more, handed out in a random order
    held, total = [_ceil(c, page) for c in cached], [_ceil(c + n, page) for c, n in zip(cached, new)]
    pages = sum(total) + sum(total) // 5 + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros((len(new), max(total) + 1), dtype=torch.int32, device=DEVICE)
    filled = held if case["kind"] == "tables" else total
    column = torch.arange(table.shape[1], device=DEVICE)[None, :]
    counts = torch.tensor(filled, device=DEVICE)[:, None]
    at = sum(filled)
    table[column < counts] = order[:at]
    s.update(table=table, held=held, total=total, pages=pages)
    if case["kind"] == "tables":
        s.update(lens=_int(cached), keep=_int(cached), new_lens=_int(new), free=order[at:].contiguous(), free_count=_int([pages - at]))
        s["free"] = torch.cat([s["free"], torch.zeros(at, dtype=torch.int32, device=DEVICE)])
        return s
    dtype = DTYPES[case["dtype"]]
    shape = (pages, case["kv_heads"], page, case["dim"])
    s["k_pages"], s["v_pages"] = _normal(gen, *shape, dtype=dtype), _normal(gen, *shape, dtype=dtype)
    s["q"] = _normal(gen, s["tokens"], case["heads"], case["dim"], dtype=dtype)
    s["kv_lens"] = _int([c + n for c, n in zip(cached, new)])
    if case["kind"] == "append":
        s["k"], s["v"] = (_normal(gen, s["tokens"], case["kv_heads"], case["dim"], dtype=dtype) for _ in range(2))
        positions = torch.cat([torch.arange(c, c + n, device=DEVICE) for c, n in zip(cached, new)])
        rows = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), torch.tensor(new, device=DEVICE))
        s["positions"] = positions.to(torch.int32)
        s["slots"] = (table[rows, positions // page] * page + positions % page).to(torch.int32)
    return s


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _run_own(s):
    from mixtral_offloading_b200 import paged_attention, paged_reserve, paged_truncate, prompt_attention, rope_append_paged
    case, kind = s["case"], s["case"]["kind"]
    if kind == "tables":
        step = paged_reserve(s["table"], s["lens"], s["free"], s["free_count"], s["new_lens"], case["page"], s["tokens"])
        dropped = paged_truncate(s["table"], s["lens"], s["free"], s["free_count"], s["keep"], case["page"])
        return [step.cu_seqlens, step.kv_lens, step.positions, step.slots, step.status, s["table"], s["lens"], s["free_count"], s["free"], dropped]
    if kind == "append":
        q = rope_append_paged(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["positions"], s["slots"], THETA)
        return [q, s["k_pages"], s["v_pages"]]
    if kind == "paged":
        return paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu_seqlens"], s["kv_lens"], s["max_new"])
    return prompt_attention(s["q"], s["k"], s["v"], s["cu_seqlens"])


# ---- their plain forms -----------------------------------------------------------------------------------------------------
def _tables(s):
    """Takes the new tokens' pages off the stack, and gives them back."""
    page, table, free = s["case"]["page"], s["table"], s["free"]
    lens, new, count = s["lens"].long(), s["new_lens"].long(), s["free_count"].long()
    after = lens + new
    first, last = (lens + page - 1) // page, (after + page - 1) // page
    need = last - first
    before = torch.cumsum(need, 0) - need
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=DEVICE), torch.cumsum(new, 0)])
    column = torch.arange(table.shape[1], device=DEVICE)[None, :]
    taken = (column >= first[:, None]) & (column < last[:, None])
    index = count - 1 - (before[:, None] + column - first[:, None])
    table.copy_(torch.where(taken, free[index.clamp(0, free.shape[0] - 1)], table))
    token = torch.arange(s["tokens"], device=DEVICE)
    row = torch.searchsorted(cu[1:], token, right=True)
    positions = lens[row] + token - cu[row]
    slots = table[row, positions // page].long() * page + positions % page
    left = count - need.sum()
    back = torch.where(taken, index, torch.full_like(index, free.shape[0]))          # every page to where it was taken from
    stack = torch.cat([free, free[:1]])
    stack.scatter_(0, back.reshape(-1), table.reshape(-1))
    free.copy_(stack[:-1])
    s["free_count"].copy_(left + need.sum())
    status = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    return [cu.to(torch.int32), after.to(torch.int32), positions.to(torch.int32), slots.to(torch.int32), status, table, s["lens"], s["free_count"],
            free, status.clone()]


def _rotate(x, turns):
    """The two halves of every head as pairs, rotated by `turns` (tokens, dim / 2) of a whole turn."""
    half = x.shape[-1] // 2
    angle = (turns - torch.round(turns)) * (2 * math.pi)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _append(s):
    page, dim = s["case"]["page"], s["case"]["dim"]
    d = torch.arange(dim // 2, device=DEVICE, dtype=torch.float64)
    turns = s["positions"].double()[:, None] * (THETA ** (-2 * d / dim) / (2 * math.pi))      # angles of far positions: 64 bits
    slots = s["slots"].long()
    s["k_pages"][slots // page, :, slots % page] = _rotate(s["k"], turns)
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    return [_rotate(s["q"], turns), s["k_pages"], s["v_pages"]]


def _attend(q, k, v, out):
    """q, out (new, heads, dim); k, v (kv_heads, length, dim): the new tokens are the last ones."""
    new, heads, dim = q.shape
    kv_heads, length, _ = k.shape
    k, v = k.float(), v.float()
    group = heads // kv_heads
    rows = max(1, (1 << 28) // (length * heads))
    for lo in range(0, new, rows):
        hi = min(new, lo + rows)
        seen = length - new + hi                                     # nothing behind it is visible to these rows
        qs = q[lo:hi].float().view(hi - lo, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * (hi - lo), dim)
        scores = (torch.matmul(qs, k[:, :seen].transpose(1, 2)) / math.sqrt(dim)).view(kv_heads, group, hi - lo, seen)
        hidden = torch.arange(seen, device=DEVICE)[None, :] > torch.arange(length - new + lo, length - new + hi, device=DEVICE)[:, None]
        scores.masked_fill_(hidden, float("-inf"))
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        total = weights.sum(-1, keepdim=True)
        mixed = torch.matmul(weights.view(kv_heads, group * (hi - lo), seen), v[:, :seen]).view(kv_heads, group, hi - lo, dim) / total
        out[lo:hi] = mixed.permute(2, 0, 1, 3).reshape(hi - lo, heads, dim).to(out.dtype)


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "tables":
        return _tables(s)
    if kind == "append":
        return _append(s)
    out = torch.empty_like(s["q"])
    for b, (lo, hi) in enumerate(zip(s["cu"], s["cu"][1:])):
        if kind == "prompt":
            k, v = s["k"][lo:hi].transpose(0, 1), s["v"][lo:hi].transpose(0, 1)
        else:
            length = s["cached"][b] + s["new"][b]
            pages = s["table"][b, :s["total"][b]].long()
            k, v = (p[pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length] for p in (s["k_pages"], s["v_pages"]))
        _attend(s["q"][lo:hi], k, v, out[lo:hi])
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    cached, new = _lengths(case)
    tokens, n = sum(new), len(new)
    if case["kind"] == "tables":
        pages = sum(_ceil(c + m, case["page"]) - _ceil(c, case["page"]) for c, m in zip(cached, new))
        # lengths and new lengths in, offsets and lengths out; a page read and written by each half; a token's position and slot
        return {"bytes": 4 * (7 * n + 4 * pages + 2 * tokens), "flops": 4 * tokens}
    q, kv = tokens * case["heads"] * case["dim"] * 2, tokens * case["kv_heads"] * case["dim"] * 2
    if case["kind"] == "append":
        return {"bytes": 2 * q + 4 * kv + 8 * tokens, "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["dim"]}
    pairs = sum(m * c + m * (m + 1) // 2 for c, m in zip(cached, new))
    flops = 4 * case["dim"] * case["heads"] * pairs
    if case["kind"] == "prompt":
        return {"bytes": 2 * q + 2 * kv + 4 * (n + 1), "flops": flops}
    length = sum(cached) + tokens
    table = 4 * sum(_ceil(c + m, case["page"]) for c, m in zip(cached, new))
    return {"bytes": 2 * q + 4 * length * case["kv_heads"] * case["dim"] + table + 8 * n, "flops": flops}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None                                                  # whole numbers
    s = prepare(case, seed)
    dim, group = case["dim"], case["heads"] // case["kv_heads"]
    if kind == "append":
        page = case["page"]
        frequency = torch.tensor([THETA ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device=DEVICE)
        angle = torch.outer(s["positions"].to(torch.float64), frequency).unsqueeze(1)
        unit = torch.polar(torch.ones_like(angle), angle)

        def turned(x):
            z = torch.complex(x[..., :dim // 2].double(), x[..., dim // 2:].double()) * unit
            return torch.cat([z.real, z.imag], dim=-1)
        keys, values, turned_keys = s["k_pages"].double(), s["v_pages"].double(), turned(s["k"])
        where = s["slots"].to(torch.int64)
        for h in range(case["kv_heads"]):
            keys[where // page, h, where % page] = turned_keys[:, h]
            values[where // page, h, where % page] = s["v"][:, h].double()
        return [turned(s["q"]), keys, values]
    if work(case)["flops"] > 1e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b in range(len(s["new"])):
        n, length, lo = s["new"][b], s["cached"][b] + s["new"][b], s["cu"][b]
        place = torch.arange(length, device=DEVICE)
        for h in range(case["heads"]):
            g = h // group
            if kind == "prompt":
                k, v = s["k"][lo:lo + n, g].double(), s["v"][lo:lo + n, g].double()
            else:
                slot = s["table"][b].long()[place // case["page"]], place % case["page"]
                k, v = s["k_pages"][slot[0], g, slot[1]].double(), s["v_pages"][slot[0], g, slot[1]].double()
            for at in range(0, n, 4096):
                q = s["q"][lo + at:lo + min(n, at + 4096), h].double()
                seen = place[None, :] <= length - n + at + torch.arange(q.shape[0], device=DEVICE)[:, None]
                logits = torch.where(seen, q @ k.T * dim ** -0.5, torch.tensor(float("-inf"), dtype=torch.float64, device=DEVICE))
                out[lo + at:lo + at + q.shape[0], h] = torch.softmax(logits, dim=-1) @ v
    return out
