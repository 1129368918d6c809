"""Keys and values of many sequences in fixed-size pages: the write of new tokens and the attention that reads them.

A cache is a pair of tensors ``[num_pages, page_size, kv_heads, head_dim]`` (views with other strides are fine, the last
dimension is contiguous).  ``page_table[b, i]`` (int32) is the page that holds positions ``i * page_size ..`` of sequence
``b``; ``seq_lens[b]`` (int32) counts its tokens *with* the new ones of the call, which are its last; the new tokens of all
sequences are packed, those of sequence ``b`` in rows ``cu_seqlens[b] : cu_seqlens[b + 1]`` (int32, as in
``flash_attention``).  A sequence may have no new tokens, rows behind the last sequence belong to none.  Lengths and
tables stay on the device: no call waits for the host, and all of them can be captured into a CUDA graph.

Bad table entries and lengths cannot be raised from the device without waiting for it.  The kernels check every page and
position themselves, touch no memory outside the cache, and record the error; ``functional.check_status()`` raises it.
The torch expressions, which run on CPU tensors, raise ``ValueError`` at once.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import check, dt, lib, ptr, sm_count, stream
from .functional import _common_dtype, _unit_inner, check_head_norm, head_norm_rope_reference, rotary_args, status_word


def _check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
                 seq_lens: torch.Tensor) -> None:
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"caches must be [num_pages, page_size, kv_heads, head_dim] of one shape and type, got "
                         f"{tuple(k_cache.shape)} {k_cache.dtype} and {tuple(v_cache.shape)} {v_cache.dtype}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("the last dimension of a cache must be contiguous")
    size = k_cache.shape[1]
    if size < 1 or size & (size - 1):
        raise ValueError(f"page_size must be a power of two, got {size}")
    if page_table.dim() != 2 or cu_seqlens.dim() != 1 or seq_lens.dim() != 1 or not (
            page_table.shape[0] == seq_lens.shape[0] == cu_seqlens.shape[0] - 1):
        raise ValueError(f"page_table [batch, pages], cu_seqlens [batch + 1] and seq_lens [batch] do not match: "
                         f"{tuple(page_table.shape)}, {tuple(cu_seqlens.shape)}, {tuple(seq_lens.shape)}")
    for name, t in (("page_table", page_table), ("cu_seqlens", cu_seqlens), ("seq_lens", seq_lens)):
        if t.dtype != torch.int32:
            raise ValueError(f"{name} must be int32, got {t.dtype}")
    if cu_seqlens.stride(0) != 1 or seq_lens.shape[0] and seq_lens.stride(0) != 1 or (
            page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("cu_seqlens, seq_lens and the rows of page_table must be contiguous")
    for name, t in (("v_cache", v_cache), ("page_table", page_table), ("cu_seqlens", cu_seqlens), ("seq_lens", seq_lens)):
        if t.device != k_cache.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {k_cache.device}")


def _check_rows(name: str, x: torch.Tensor, k_cache: torch.Tensor) -> None:
    if x.dim() != 3 or x.shape[2] != k_cache.shape[3] or x.dtype != k_cache.dtype or x.device != k_cache.device:
        raise ValueError(f"{name} {tuple(x.shape)} {x.dtype} {x.device} does not fit a cache "
                         f"{tuple(k_cache.shape)} {k_cache.dtype} {k_cache.device}")


def _no_grad_inputs(what: str, *ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise _lib.KernelError(f"{what} has no backward pass: call it under torch.no_grad()")


def _token_places(page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, tokens: int,
                  page_size: int, num_pages: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(row, position, page, slot) of the new tokens that belong to a sequence; raises on a token without a place."""
    rows, places = [], []
    cu, lens = cu_seqlens.tolist(), seq_lens.tolist()
    for b, length in enumerate(lens):
        start, end = max(cu[b], 0), min(cu[b + 1], tokens)
        rows.extend(range(start, end))
        places.extend((b, length - cu[b + 1] + t) for t in range(start, end))
    row = torch.tensor(rows, dtype=torch.int64)
    seq = torch.tensor([b for b, _ in places], dtype=torch.int64)
    pos = torch.tensor([p for _, p in places], dtype=torch.int64)
    if pos.numel() and (int(pos.min()) < 0 or int(pos.max()) >= page_table.shape[1] * page_size):
        raise ValueError("a new token lies outside its sequence's page table")
    page = page_table[seq, pos // page_size].to(torch.int64)
    if page.numel() and (int(page.min()) < 0 or int(page.max()) >= num_pages):
        raise ValueError("a new token lies in a page outside the cache")
    return row, pos, page, pos % page_size


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor,
                 q: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, q_bias: Optional[torch.Tensor] = None,
                 k_bias: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                 rotary: Optional[tuple[int, float, bool]] = None, eps: float = 1e-5,
                 rms: bool = True) -> Optional[torch.Tensor]:
    """Write the keys and values of new tokens into their pages; keys (and queries, if given) pass the per-head norm and
    the rotary embedding of ``functional.qk_norm_rope`` on the way.  Returns the queries as a new tensor, or None.

    ``k, v [tokens, kv_heads, d]`` and ``q [tokens, heads, d]`` are projections with any strides.  Without weights there
    is no norm, without ``rotary`` no rotation (keys are then copied bit by bit).  Angles follow each token's place in
    its sequence, or ``positions`` (int32 ``[tokens]``).  No page may be named twice among the places written.  Rows
    behind the last sequence touch no page and give zero queries.  In inference only: no backward pass."""
    _check_cache(k_cache, v_cache, page_table, cu_seqlens, seq_lens)
    _no_grad_inputs("paged_append", k, v, q, q_weight, k_weight, q_bias, k_bias, k_cache, v_cache)
    for name, x in (("k", k), ("v", v)):
        _check_rows(name, x, k_cache)
        if x.shape[:2] != (k.shape[0], k_cache.shape[2]):
            raise ValueError(f"{name} {tuple(x.shape)} does not match {k.shape[0]} tokens of {k_cache.shape[2]} kv heads")
    check_head_norm("k", k, k_weight, k_bias, rms)
    if q is not None:
        _check_rows("q", q, k_cache)
        check_head_norm("q", q, q_weight, q_bias, rms)
        if q.shape[0] != k.shape[0]:
            raise ValueError(f"q has {q.shape[0]} tokens, k {k.shape[0]}")
    elif q_weight is not None or q_bias is not None:
        raise ValueError("norm parameters for queries without queries")
    rot, base, interleaved = rotary_args(rotary, k.shape[2])
    if positions is not None and (positions.shape != (k.shape[0],) or positions.dtype != torch.int32
                                  or positions.device != k.device or not positions.is_contiguous()):
        raise ValueError(f"positions must be contiguous int32 [{k.shape[0]}] on {k.device}")
    tokens, kv_heads, d = k.shape
    num_pages, page_size = k_cache.shape[:2]
    if not k.is_cuda:
        row, pos, page, slot = _token_places(page_table, cu_seqlens, seq_lens, tokens, page_size, num_pages)
        pos = pos if positions is None else positions[row].to(torch.int64)
        k_cache[page, slot] = head_norm_rope_reference(k[row], k_weight, k_bias, pos, rotary, eps, rms)
        v_cache[page, slot] = v[row]
        if q is None:
            return None
        out = torch.zeros(q.shape, dtype=q.dtype)
        out[row] = head_norm_rope_reference(q[row], q_weight, q_bias, pos, rotary, eps, rms)
        return out
    if d > 256:
        raise _lib.KernelError(f"paged_append: head size {d} is not supported (up to 256)")
    code = dt(k.dtype)
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if tokens == 0:
        return out
    k, v = _unit_inner(k), _unit_inner(v)
    q = None if q is None else _unit_inner(q)
    wq, wk, bq, bk = _common_dtype(q_weight, k_weight, q_bias, k_bias)
    w_code = next((dt(w.dtype) for w in (wq, wk) if w is not None), 0)
    with _lib.on_device_of(k):
        check(lib().sb200_paged_append(
            ptr(q), k.data_ptr(), v.data_ptr(), ptr(out), k_cache.data_ptr(), v_cache.data_ptr(), ptr(wq), ptr(wk),
            ptr(bq), ptr(bk), ptr(positions), page_table.data_ptr(), cu_seqlens.data_ptr(), seq_lens.data_ptr(), tokens,
            seq_lens.shape[0], 0 if q is None else q.shape[1], kv_heads, d, 0 if q is None else q.stride(0),
            0 if q is None else q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), k_cache.stride(0),
            k_cache.stride(1), k_cache.stride(2), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            page_table.stride(0), page_table.shape[1], num_pages, page_size, float(eps), int(rms), rot, base,
            int(interleaved), code, w_code, sm_count(), status_word().data_ptr(), stream()), "sb200_paged_append")
    return out
