"""Attention over the paged cache outside the page selection: sliding window with
first tokens kept visible, and decode of a batch that shares long prefixes (host
wrappers of ``locks_window_attention`` and ``locks_shared_prefix_decode``).

A query row with a seen score of NaN or +inf becomes NaN; keys and values must be
finite.  Weights are rounded to bf16 in the product with V where a request has more
than 16 rows (query tokens x G) and over a shared prefix, else carried to 2^-17.

Caches come in either engine layout, (NB, 2, page, n_kv, d) or (2, NB, page, n_kv, d),
with any strides whose rows are 16-byte aligned and whose head stride is a multiple
of 64 (a head-major view too); one of exactly two blocks is read as the latter."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi
from .decode import _planes

NO_WINDOW = 2 ** 31 - 1      # larger counts than the entry point's integers hold mean all


def _checked(q, kv_cache, block_table, out, lse, scratch, status, n_kv, G, ints):
    """What both calls check of their tensors; the arguments both pass on."""
    k, v, (n_blocks, page, heads, d), cs = _planes(kv_cache)
    bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    assert q.dtype is bf16 and out.dtype is bf16 and kv_cache.dtype is bf16
    shape, qs, os = q.shape, q.stride(), out.stride()
    assert len(shape) == 3 and out.shape == shape
    assert shape[1] == n_kv * G and heads == n_kv and shape[2] == d
    assert qs[2] == os[2] == cs[3] == 1
    bs = block_table.stride()
    assert block_table.dtype is i32 and bs[1] == 1
    for t in ints:
        assert t.dtype is i32 and t.is_contiguous(), \
            "lengths and bounds are contiguous int32"
    assert status is None or status.dtype is i32, "status is int32"
    lse_at, lse_stride, scratch_at, floats = None, 0, None, 0
    if lse is not None:
        lse_stride, one = lse.stride()
        assert lse.dtype is f32 and one == 1 and lse.shape == shape[:2]
        lse_at = lse.data_ptr()
    if scratch is not None:
        assert scratch.dtype is f32 and scratch.is_contiguous()
        scratch_at, floats = scratch.data_ptr(), scratch.numel()
    return ((q.data_ptr(), qs[0], qs[1], k, v, cs[0], cs[1], cs[2],
             block_table.data_ptr(), bs[0], block_table.shape[1], n_blocks),
            (out.data_ptr(), os[0], os[1], lse_at, lse_stride, scratch_at, floats),
            d, page)


def window_paged_attention(q: torch.Tensor, kv_cache: torch.Tensor,
                           block_table: torch.Tensor, cu_q: torch.Tensor,
                           seq_lens: torch.Tensor, out: torch.Tensor, *, n_kv: int,
                           G: int, window: Optional[int], sinks: int = 0,
                           scale: float, max_q: int,
                           scratch: Optional[torch.Tensor] = None,
                           lse: Optional[torch.Tensor] = None,
                           status: Optional[torch.Tensor] = None) -> None:
    """Attention of ragged query runs; writes ``out`` (and ``lse``) in place.

    Request r's queries are rows ``cu_q[r] : cu_q[r + 1]`` of q (T, H, d); it has
    ``seq_lens[r]`` tokens in the cache, the new ones among them.  A query at
    position p sees keys j <= p with p - j < ``window`` or j < ``sinks``
    (``window`` None: all of them).  Rows that see nothing become 0 (lse -inf),
    rows behind ``cu_q[R]`` stay as they were, pages that nobody sees are not read.
    ``max_q``: the query tokens of the longest request; it steers how the work is cut,
    a request with more is answered all the same, more slowly (0: nothing is done).
    ``scratch``: fp32 workspace that lets the long keys of few queries be cut into
    parts, see :func:`attention_scratch_floats` (the default of two parts is not enough
    for single tokens); calls that may overlap on the GPU need one each.  ``status``:
    int32, set where a bounded wait ran out."""
    dev = _cabi.one_device(q, kv_cache, block_table, cu_q, seq_lens, out, scratch, lse,
                           status)
    source, target, d, page = _checked(q, kv_cache, block_table, out, lse, scratch,
                                       status, n_kv, G, (cu_q, seq_lens))
    R = seq_lens.numel()
    assert cu_q.numel() == R + 1 and block_table.shape[0] == R
    if R == 0 or q.shape[0] == 0:
        return
    _cabi.call_on(dev, "locks_window_attention", *source, cu_q.data_ptr(),
                  seq_lens.data_ptr(), *target, q.shape[0], R, min(max_q, NO_WINDOW), n_kv,
                  G, d, page, NO_WINDOW if window is None else min(window, NO_WINDOW),
                  min(sinks, NO_WINDOW), scale, _cabi.addr(status))


def shared_prefix_paged_decode(q: torch.Tensor, kv_cache: torch.Tensor,
                               block_table: torch.Tensor, seq_lens: torch.Tensor,
                               cu_groups: torch.Tensor, prefix_lens: torch.Tensor,
                               out: torch.Tensor, *, n_kv: int, G: int, scale: float,
                               scratch: torch.Tensor,
                               lse: Optional[torch.Tensor] = None,
                               status: Optional[torch.Tensor] = None) -> None:
    """One query token per request, q (R, H, d), over all its ``seq_lens[r]``
    cached tokens; the requests ``cu_groups[g] : cu_groups[g + 1]`` have the first
    ``prefix_lens[g]`` tokens in common and those are read once for the group
    (through the table row of its first request).  Writes ``out`` (and ``lse``) in
    place; rows outside the groups stay as they were.  ``scratch``: fp32 workspace,
    at least ``attention_scratch_floats(R, H, d)`` elements."""
    dev = _cabi.one_device(q, kv_cache, block_table, seq_lens, cu_groups, prefix_lens,
                           out, scratch, lse, status)
    source, target, d, page = _checked(q, kv_cache, block_table, out, lse, scratch,
                                       status, n_kv, G, (seq_lens, cu_groups, prefix_lens))
    R, groups = q.shape[0], prefix_lens.numel()
    assert seq_lens.numel() == block_table.shape[0] == R
    assert cu_groups.numel() == groups + 1
    if R == 0 or groups == 0:
        return
    _cabi.call_on(dev, "locks_shared_prefix_decode", *source, seq_lens.data_ptr(),
                  cu_groups.data_ptr(), prefix_lens.data_ptr(), *target, R, groups,
                  n_kv, G, d, page, scale, _cabi.addr(status))


def attention_scratch_floats(n_rows: int, n_heads: int, head_dim: int = 128,
                             parts: int = 2) -> int:
    """fp32 elements that ``parts`` partial results of ``n_rows`` query tokens take
    (a maximum, a sum and ``head_dim`` values per head).  Shared-prefix decode needs
    two; up to SMs / n_kv + 1 of them are of use to it.  A windowed call uses two or
    more where a request has over 16 rows (tokens x G), and four or more, up to 2 * SMs
    / (requests * n_kv), for single tokens and the like over 2048 pages or more."""
    return int(n_rows) * int(n_heads) * (int(head_dim) + 2) * int(parts)
