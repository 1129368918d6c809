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

import math
from typing import Optional

import torch

from . import _lib
from ._lib import check, dt, lib, ptr, sm_count, stream
from .functional import _common_dtype, _unit_inner, argument_word, check_head_norm, head_norm_rope_reference, rotary_args


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


def _check_sizes(what: str, *sizes: int) -> None:
    if any(s >= 2 ** 31 - 2 ** 16 for s in sizes):
        raise _lib.KernelError(f"{what}: sizes {sizes} pass 32 bits")


def _refuse_shared_memory(name: str, t: torch.Tensor) -> None:
    """Written tensors need memory of their own for every element (sufficient: each stride spans the smaller ones)."""
    if t.is_contiguous():
        return
    span = 1
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if stride < span:
            raise ValueError(f"elements of {name} share memory: shape {tuple(t.shape)} with strides {t.stride()}")
        span += stride * (size - 1)


def _check_rows(name: str, x: torch.Tensor, k_cache: torch.Tensor) -> None:
    if x.dim() != 3 or x.shape[2] != k_cache.shape[3] or x.dtype != k_cache.dtype or x.device != k_cache.device:
        raise ValueError(f"{name} {tuple(x.shape)} {x.dtype} {x.device} does not fit a cache "
                         f"{tuple(k_cache.shape)} {k_cache.dtype} {k_cache.device}")


def _no_grad_inputs(what: str, *ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise _lib.KernelError(f"{what} has no backward pass: call it under torch.no_grad()")


def _row_ends(cu_seqlens: torch.Tensor, tokens: int) -> list[int]:
    cu = cu_seqlens.tolist()
    if any(not 0 <= a <= b <= tokens for a, b in zip(cu, cu[1:])):
        raise ValueError(f"cu_seqlens {cu} do not follow one another inside {tokens} rows")
    return cu


def _token_places(page_table: torch.Tensor, cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, tokens: int,
                  page_size: int, num_pages: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(row, position, page, slot) of the new tokens that belong to a sequence; raises on a token without a place."""
    rows, places = [], []
    cu, lens = _row_ends(cu_seqlens, tokens), seq_lens.tolist()
    for b, length in enumerate(lens):
        start, end = cu[b], cu[b + 1]
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
    _refuse_shared_memory("k_cache", k_cache)
    _refuse_shared_memory("v_cache", v_cache)
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
    _check_sizes("paged_append", tokens, num_pages, page_table.shape[0], page_table.shape[1], page_size)
    code = dt(k.dtype)
    out = None if q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
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
            int(interleaved), code, w_code, sm_count(), argument_word().data_ptr(), stream()), "sb200_paged_append")
    return out


def paged_attention_reference(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                              cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, causal: bool, scale: float,
                              window: Optional[int], out: torch.Tensor) -> torch.Tensor:
    """Sequence by sequence in fp32 (fp64 for fp64 inputs); raises on visible pages outside the cache."""
    size, kv_heads = k_cache.shape[1], k_cache.shape[2]
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    group = q.shape[1] // kv_heads
    cu = _row_ends(cu_seqlens, q.shape[0])
    for b, length in enumerate(seq_lens.tolist()):
        start, end = cu[b], cu[b + 1]
        n = end - start
        if n == 0:
            continue
        if not 0 <= length <= page_table.shape[1] * size:
            raise ValueError(f"sequence {b} has length {length}, its page table {page_table.shape[1] * size} places")
        pos = torch.arange(length - n, length, device=q.device)
        lo = torch.zeros_like(pos) if window is None else (pos - window).clamp_(min=0)
        hi = pos + 1 if causal else torch.full_like(pos, length)
        if window is not None and not causal:
            hi = torch.minimum(hi, pos + window + 1)
        first, last = int(lo.min()) // size, -(-max(int(hi.max()), 0) // size)
        pages = page_table[b, first:last].to(torch.int64)
        if pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= k_cache.shape[0]):
            raise ValueError(f"sequence {b} sees a page outside the cache")
        j = torch.arange(first * size, max(min(last * size, length), first * size), device=q.device)
        seen = (j[None] >= lo[:, None]) & (j[None] < hi[:, None])  # [n, keys]
        k, v = (c[pages].reshape(-1, kv_heads, c.shape[3])[:j.numel()].to(acc) for c in (k_cache, v_cache))
        v = v.masked_fill(~seen.any(0)[:, None, None], 0.0)
        qs = q[start:end].reshape(n, kv_heads, group, -1).to(acc)
        s = torch.einsum("nhgd,jhd->hgnj", qs, k).mul_(scale).masked_fill_(~seen, float("-inf"))
        p = torch.softmax(s, -1).masked_fill(~seen.any(1)[:, None], 0.0)
        out[start:end] = torch.einsum("hgnj,jhd->nhgd", p, v).reshape(n, q.shape[1], -1).to(q.dtype)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    cu_seqlens: torch.Tensor, seq_lens: torch.Tensor, causal: bool = True,
                    scale: Optional[float] = None, window: Optional[int] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the new tokens ``q [tokens, heads, d]`` of many sequences over their cached keys and values, one token
    or a long chunk each; returns ``[tokens, heads, d]`` (``out``, if given).

    Heads are a multiple of the cache's KV heads.  A query at position ``i`` of its sequence sees the cached positions
    ``j <= i`` (all of them without ``causal``) with ``|i - j| <= window``; keys of the new tokens are read from the
    cache, so they are written first (``paged_append``).  A query that sees nothing gives zeros.  Pages that no query of
    the call sees may be missing from the table.  Rows of no sequence are left as they were in ``out`` and are zero
    without it; ``out`` may be ``q`` itself and overlaps no other tensor.  Whatever the cache holds behind a sequence's
    last token has no effect; keys and values of its tokens are finite.  On GPUs: bf16 and fp16 (probabilities are rounded
    to that type, sums are not), head sizes that are multiples of 8 up to 128, pages of 8 tokens and more, page tables of up
    to 2^26 positions, 2^17 sequences, 2^30 query rows and 2^15 heads per KV head; products of 256 rows (64 in decoding)
    with 128 keys, and four more for each block of rows, add up to less than 2^31 (else zeros and an error that
    ``check_status`` raises).  In inference only: no backward pass."""
    _check_cache(k_cache, v_cache, page_table, cu_seqlens, seq_lens)
    _no_grad_inputs("paged_attention", q, k_cache, v_cache, out)
    _check_rows("q", q, k_cache)
    tokens, heads, d = q.shape
    num_pages, page_size, kv_heads = k_cache.shape[:3]
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are not a multiple of {kv_heads} kv heads")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"the softmax scale must be positive and finite, got {scale}")
    if window is not None and window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} {out.device} does not match q {tuple(q.shape)} {q.dtype}")
    if out is not None:
        _refuse_shared_memory("out", out)
    if not q.is_cuda:
        return paged_attention_reference(q, k_cache, v_cache, page_table, cu_seqlens, seq_lens, causal, scale, window,
                                         torch.zeros_like(q) if out is None else out)
    if q.dtype not in (torch.bfloat16, torch.float16) or d % 8 or not 8 <= d <= 128 or page_size < 8:
        raise _lib.KernelError(f"paged_attention: {q.dtype} with head size {d} and pages of {page_size} is not supported "
                               "(bf16 / fp16, multiples of 8 up to 128, pages of 8 and more)")
    zero_tail = out is None
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.numel() == 0:
        return out
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("out", out)):
        if t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:-1]) or t.data_ptr() % 16:
            raise _lib.KernelError(f"paged_attention: {name} must start and have its rows on 16-byte boundaries, strides "
                                   f"{t.stride()}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if num_pages > 1 and (t.stride(1) <= 0 or t.stride(0) % (8 * t.stride(1))):
            raise _lib.KernelError(f"paged_attention: the page stride of {name} must be a multiple of eight row strides, "
                                   f"got {t.stride()}")
    if num_pages == 0:
        raise ValueError("the cache has no pages")
    _check_sizes("paged_attention", tokens * heads, num_pages, page_table.shape[0], page_table.shape[1], page_size)
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # also where only the start is off
    with _lib.on_device_of(q):
        batch, cols, sms = seq_lens.shape[0], page_table.shape[1], sm_count()
        size = lib().sb200_paged_attention_workspace(tokens, batch, heads, kv_heads, d, cols * page_size, sms)
        workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        check(lib().sb200_paged_attention(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), page_table.data_ptr(),
            cu_seqlens.data_ptr(), seq_lens.data_ptr(), workspace.data_ptr(), size, tokens, batch, heads, kv_heads, d,
            num_pages, page_size, cols, page_table.stride(0), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
            k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), v_cache.stride(0), v_cache.stride(1),
            v_cache.stride(2), int(causal), -1 if window is None else min(int(window), 2 ** 30), scale, int(zero_tail),
            dt(q.dtype), sms, argument_word().data_ptr(), stream()), "sb200_paged_attention")
    return out
