"""A key/value cache in pages, and the attention that reads it: sequences of different lengths in one pool, prompts that
arrive in chunks beside running generations.

The reference generates through Hugging Face (src/build_model.py:166-241 assembles the model), whose cache is one tensor per
layer and batch.  Here a layer's keys, and its values, are (pages, n_kv_heads, page_size, head_dim); block_table (sequences,
max_pages) int32 names the pages of every sequence, kv_lens (sequences,) int32 how many positions it has.  A step is

    step = paged_reserve(block_table, kv_lens, free_pages, free_count, new_lens, page_size, tokens)
    q = rope_append_paged(q, k, v, k_pages, v_pages, step.positions, step.slots, theta)          # every layer
    out = paged_attention(q, k_pages, v_pages, block_table, step.cu_seqlens, step.kv_lens, max_new)

None of them reads a length on the host, so that a captured graph follows the lengths in device memory.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _cabi

_CODES = {torch.bfloat16: 0, torch.float16: 1}


class PagedStep(NamedTuple):
    """What paged_reserve leaves for a step's operators (all int32, on the device)."""
    cu_seqlens: torch.Tensor     # (sequences + 1,): first row of every sequence among the new tokens
    kv_lens: torch.Tensor        # (sequences,): lengths with the new tokens
    positions: torch.Tensor      # (tokens,), -1 behind the last token
    slots: torch.Tensor          # (tokens,): page * page_size + row in the page, -1 behind the last token
    status: torch.Tensor         # (1,): 0, or why nothing was reserved (hqm_paged_reserve)


def _ints(device, **tensors) -> None:
    for name, t in tensors.items():
        if t.device != device or t.dtype != torch.int32:
            raise ValueError(f"{name} has to be int32 on {device}, not {t.dtype} on {t.device}")
        if t.dim() > 0 and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} has to be contiguous")


def _tables(block_table, kv_lens, free_pages, free_count, lens, name):
    _cabi.require_cuda(block_table)
    _ints(block_table.device, block_table=block_table, kv_lens=kv_lens, free_pages=free_pages, free_count=free_count, **{name: lens})
    if block_table.dim() != 2 or free_pages.dim() != 1 or free_count.numel() != 1:
        raise ValueError("block_table is (sequences, max_pages), free_pages a vector, free_count one number")
    B = block_table.shape[0]
    if kv_lens.shape != (B,) or lens.shape != (B,):
        raise ValueError(f"{B} sequences in the table, kv_lens {tuple(kv_lens.shape)}, {name} {tuple(lens.shape)}")
    return B, block_table.shape[1], block_table.stride(0) if B > 1 else block_table.shape[1]


def paged_reserve(block_table: torch.Tensor, kv_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  new_lens: torch.Tensor, page_size: int, tokens: int) -> PagedStep:
    """new_lens[b] more positions for every sequence b, in one launch (hqm_paged_reserve): pages come off the stack
    free_pages[: free_count], block_table, kv_lens and free_count are updated in place.  `tokens`: rows of the step (at least
    the sum of new_lens; the rows behind it get position and slot -1).  All or nothing: with a status other than 0 the
    cache is as it was and the step has no tokens."""
    step = _cabi.host().paged_reserve(block_table, kv_lens, free_pages, free_count, new_lens, page_size, tokens)
    if step is not None:
        return PagedStep(*step)
    B, max_pages, stride = _tables(block_table, kv_lens, free_pages, free_count, new_lens, "new_lens")
    if tokens < 0:
        raise ValueError(f"a step of {tokens} tokens")
    dev = block_table.device
    cu, after, positions, slots, status = torch.empty(2 * B + 2 + 2 * tokens, dtype=torch.int32, device=dev).split(
        (B + 1, B, tokens, tokens, 1))
    with torch.cuda.device(dev):
        _cabi.check(_cabi.lib().hqm_paged_reserve(
            _cabi.ptr(block_table), stride, _cabi.ptr(kv_lens), _cabi.ptr(free_pages), _cabi.ptr(free_count), _cabi.ptr(new_lens),
            _cabi.ptr(cu), _cabi.ptr(after), _cabi.ptr(positions), _cabi.ptr(slots), _cabi.ptr(status), B, max_pages, page_size,
            free_pages.shape[0], tokens, _cabi.stream_ptr(dev)))
    return PagedStep(cu, after, positions, slots, status)


def paged_truncate(block_table: torch.Tensor, kv_lens: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                   keep: torch.Tensor, page_size: int) -> torch.Tensor:
    """Every sequence keeps its first keep[b] positions, the pages behind them go back on the stack (hqm_paged_truncate).
    Returns the status (1,): 0, or why nothing changed."""
    status = _cabi.host().paged_truncate(block_table, kv_lens, free_pages, free_count, keep, page_size)
    if status is not None:
        return status
    B, max_pages, stride = _tables(block_table, kv_lens, free_pages, free_count, keep, "keep")
    dev = block_table.device
    status = torch.empty(1, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _cabi.check(_cabi.lib().hqm_paged_truncate(
            _cabi.ptr(block_table), stride, _cabi.ptr(kv_lens), _cabi.ptr(free_pages), _cabi.ptr(free_count), _cabi.ptr(keep),
            _cabi.ptr(status), B, max_pages, page_size, free_pages.shape[0], _cabi.stream_ptr(dev)))
    return status


def _strides(t: torch.Tensor):
    """Strides of (tokens, heads, head_dim) in elements (of a dimension of one: what a contiguous tensor has)."""
    token = t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]
    head = t.stride(1) if t.shape[1] > 1 else t.shape[2]
    return token, head


def _heads(q: torch.Tensor, **others) -> int:
    """Checks types, devices and the last dimension; the code of the type."""
    _cabi.require_cuda(q)
    if q.dtype not in _CODES:
        raise ValueError(f"bf16 or fp16, not {q.dtype}")
    for name, t in dict(q=q, **others).items():
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, q {q.dtype} on {q.device}")
        if t.shape[-1] != q.shape[-1] or (t.shape[-1] > 1 and t.stride(-1) != 1):
            raise ValueError(f"{name}: rows of {q.shape[-1]} contiguous elements, not {tuple(t.shape)} with strides {t.stride()}")
    return _CODES[q.dtype]


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError(f"pages are (pages, n_kv_heads, page_size, head_dim), not {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    pages, n_kv, page_size, dim = k_pages.shape
    for t in (k_pages, v_pages):
        if (page_size > 1 and t.stride(2) != dim) or (n_kv > 1 and t.stride(1) != page_size * dim):
            raise ValueError("a page has to be contiguous (pages may lie apart)")
    one = n_kv * page_size * dim
    return pages, n_kv, page_size, k_pages.stride(0) if pages > 1 else one, v_pages.stride(0) if pages > 1 else one


def _out(q: torch.Tensor, out: Optional[torch.Tensor], name: str = "out") -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
        raise ValueError(f"{name} has to be contiguous, {tuple(q.shape)} {q.dtype} on {q.device}")
    return out


def rope_append_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      positions: torch.Tensor, slots: torch.Tensor, theta: float, out: Optional[torch.Tensor] = None,
                      k_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of q (T, n_heads, head_dim) and k (T, n_kv_heads, head_dim) at `positions` (T,), and append of k and v
    to the pages at `slots` (T,), in one launch (hqm_rope_append_paged).  Returns the rotated q: `out`, which may be q itself, or
    a new tensor; k_out, which may be k itself, receives the rotated k as well (prompt_attention wants it).  Tokens with a
    negative slot are left out (their rows of `out` and `k_out` stay as they were; of a new tensor they are not initialised).
    No two tokens may have the same slot.
    Otherwise what is written shares no memory with what is read, nor keys with values (ValueError).  Angles in 64 bits, one rounding."""
    done = _cabi.host().rope_append_paged(q, k, v, k_pages, v_pages, positions, slots, theta, out, k_out)
    if done is not None:
        return done
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0]:
        raise ValueError(f"q (T, n_heads, head_dim), k and v (T, n_kv_heads, head_dim), not {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    code = _heads(q, k=k, v=v, k_pages=k_pages, v_pages=v_pages)
    pages, n_kv, page_size, k_page, v_page = _pool(k_pages, v_pages)
    T, n_heads, dim = q.shape
    if k.shape[1] != n_kv:
        raise ValueError(f"{k.shape[1]} key/value heads, {n_kv} in the pages")
    _ints(q.device, positions=positions, slots=slots)
    if positions.shape != (T,) or slots.shape != (T,):
        raise ValueError(f"positions and slots of {T} tokens, not {tuple(positions.shape)} and {tuple(slots.shape)}")
    out = _out(q, out)
    if k_out is not None:
        _out(k, k_out, "k_out")
    high = C.c_float(theta).value
    call = _cabi.HqmPagedAppend(
        out.data_ptr(), None if k_out is None else k_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v), k_pages.data_ptr(),
        v_pages.data_ptr(), k_page, v_page, positions.data_ptr(), slots.data_ptr(), T, n_heads, n_kv, dim, pages, page_size, code, high, theta - high)
    with torch.cuda.device(q.device):
        _cabi.check(_cabi.lib().hqm_rope_append_paged(C.byref(call), _cabi.stream_ptr(q.device)))
    return out


def _attention(entry, call, q):
    lib = _cabi.lib()
    with torch.cuda.device(q.device):
        need = lib.hqm_attention_scratch_bytes(C.byref(call))
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        _cabi.check(getattr(lib, entry)(C.byref(call), _cabi.ptr(ws), need, _cabi.stream_ptr(q.device)))


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, cu_seqlens: torch.Tensor,
                    kv_lens: torch.Tensor, max_new: int, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens of many sequences over their pages (hqm_paged_attention): q (T, n_heads, head_dim), sequence
    b's rows are cu_seqlens[b] .. cu_seqlens[b + 1] - 1, and its kv_lens[b] positions, the new tokens' last among them, are in the
    pages already.  New token i of n sees positions 0 .. kv_lens[b] - n + i; a row that sees nothing is 0.  max_new: no sequence
    has more new tokens (1 for a decoding step).  scale: 1 / sqrt(head_dim) unless given.  Rows behind the last sequence are
    left as they were in `out` (of a new tensor they are not initialised), which shares no memory with q or the pages."""
    done = _cabi.host().attention(q, k_pages, v_pages, cu_seqlens, max_new, scale, out, block_table, kv_lens)
    if done is not None:
        return done
    if q.dim() != 3:
        raise ValueError(f"q is (T, n_heads, head_dim), not {tuple(q.shape)}")
    code = _heads(q, k_pages=k_pages, v_pages=v_pages)
    pages, n_kv, page_size, k_page, v_page = _pool(k_pages, v_pages)
    T, n_heads, dim = q.shape
    _ints(q.device, block_table=block_table, cu_seqlens=cu_seqlens, kv_lens=kv_lens)
    B = kv_lens.shape[0]
    if block_table.dim() != 2 or block_table.shape[0] != B or cu_seqlens.shape != (B + 1,) or kv_lens.dim() != 1:
        raise ValueError(f"block_table (B, max_pages), cu_seqlens (B + 1,), kv_lens (B,), not {tuple(block_table.shape)}, "
                         f"{tuple(cu_seqlens.shape)}, {tuple(kv_lens.shape)}")
    out = _out(q, out)
    call = _cabi.HqmAttention(
        out.data_ptr(), q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), *_strides(q), 0, 0, 0, 0, k_page, v_page,
        block_table.data_ptr(), block_table.stride(0) if B > 1 else block_table.shape[1], cu_seqlens.data_ptr(), kv_lens.data_ptr(), T, B,
        max_new, n_heads, n_kv, dim, pages, page_size, block_table.shape[1], code, dim ** -0.5 if scale is None else scale)
    _attention("hqm_paged_attention", call, q)
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, max_len: Optional[int] = None,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over whole prompts, packed one behind the other (hqm_prompt_attention): q (T, n_heads, head_dim), k and v
    (T, n_kv_heads, head_dim), sequence b's rows are cu_seqlens[b] .. cu_seqlens[b + 1] - 1.  max_len: no prompt is longer (T
    unless given).  scale and out as for paged_attention."""
    done = _cabi.host().attention(q, k, v, cu_seqlens, q.shape[0] if max_len is None else max_len, scale, out)
    if done is not None:
        return done
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[0] != k.shape[0]:
        raise ValueError(f"q (T, n_heads, head_dim), k and v (T, n_kv_heads, head_dim), not {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    code = _heads(q, k=k, v=v)
    T, n_heads, dim = q.shape
    _ints(q.device, cu_seqlens=cu_seqlens)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError(f"cu_seqlens is (B + 1,), not {tuple(cu_seqlens.shape)}")
    out = _out(q, out)
    call = _cabi.HqmAttention(
        out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), *_strides(q), *_strides(k), *_strides(v), 0, 0, None, 0,
        cu_seqlens.data_ptr(), None, T, cu_seqlens.shape[0] - 1, T if max_len is None else max_len, n_heads, k.shape[1], dim, 0, 0, 0, code,
        dim ** -0.5 if scale is None else scale)
    _attention("hqm_prompt_attention", call, q)
    return out
