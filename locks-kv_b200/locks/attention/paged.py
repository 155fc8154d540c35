"""Attention over the paged cache outside the page selection: sliding window with
first tokens kept visible, and decode of a batch that shares long prefixes (host
wrappers of ``locks_window_attention`` and ``locks_shared_prefix_decode``)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi
from .decode import _split_kv

NO_WINDOW = 2 ** 31 - 1


def _checked(q, kv_cache, block_table, out, lse, n_kv, G, ints):
    k, v = _split_kv(kv_cache)
    assert v is not None, "the cache has no V half"
    bf16 = torch.bfloat16
    assert q.dtype == out.dtype == k.dtype == bf16
    assert q.dim() == 3 and q.shape[1] == n_kv * G and out.shape == q.shape
    assert q.stride(2) == out.stride(2) == k.stride(3) == v.stride(3) == 1
    assert k.stride() == v.stride(), "K and V planes must share strides"
    assert k.shape[2] == n_kv and k.shape[3] == q.shape[2]
    assert block_table.dtype == torch.int32 and block_table.stride(1) == 1
    for t in ints:
        assert t.dtype == torch.int32 and t.is_contiguous(), \
            "lengths and bounds are contiguous int32"
    if lse is not None:
        assert lse.dtype == torch.float32 and lse.stride(1) == 1
        assert lse.shape == q.shape[:2]
    return k, v


def _scratch(scratch):
    if scratch is None:
        return 0
    assert scratch.dtype == torch.float32 and scratch.is_contiguous()
    return scratch.numel()


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
    ``max_q`` bounds the query tokens of a request.  ``scratch``: fp32 workspace
    for long keys with few queries, see :func:`attention_scratch_floats`; calls
    that may overlap on the GPU need one each."""
    k, v = _checked(q, kv_cache, block_table, out, lse, n_kv, G, (cu_q, seq_lens))
    dev = _cabi.one_device(q, kv_cache, block_table, cu_q, seq_lens, out, scratch, lse,
                           status)
    R = seq_lens.shape[0]
    assert cu_q.shape[0] == R + 1 and block_table.shape[0] == R
    _cabi.call_on(dev, "locks_window_attention", _cabi.ptr(q), q.stride(0), q.stride(1),
                  _cabi.ptr(k), _cabi.ptr(v), k.stride(0), k.stride(1), k.stride(2),
                  _cabi.ptr(block_table), block_table.stride(0), block_table.shape[1],
                  k.shape[0], _cabi.ptr(cu_q), _cabi.ptr(seq_lens), _cabi.ptr(out),
                  out.stride(0), out.stride(1), _cabi.ptr(lse),
                  lse.stride(0) if lse is not None else 0, _cabi.ptr(scratch),
                  _scratch(scratch), q.shape[0], R, int(max_q), int(n_kv), int(G),
                  q.shape[2], k.shape[1],
                  NO_WINDOW if window is None else min(int(window), NO_WINDOW),
                  int(sinks), float(scale), _cabi.ptr(status))


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
    k, v = _checked(q, kv_cache, block_table, out, lse, n_kv, G,
                    (seq_lens, cu_groups, prefix_lens))
    dev = _cabi.one_device(q, kv_cache, block_table, seq_lens, cu_groups, prefix_lens,
                           out, scratch, lse, status)
    R = q.shape[0]
    assert seq_lens.shape[0] == block_table.shape[0] == R
    assert cu_groups.shape[0] == prefix_lens.shape[0] + 1
    _cabi.call_on(dev, "locks_shared_prefix_decode", _cabi.ptr(q), q.stride(0),
                  q.stride(1), _cabi.ptr(k), _cabi.ptr(v), k.stride(0), k.stride(1),
                  k.stride(2), _cabi.ptr(block_table), block_table.stride(0),
                  block_table.shape[1], k.shape[0], _cabi.ptr(seq_lens),
                  _cabi.ptr(cu_groups), _cabi.ptr(prefix_lens), _cabi.ptr(out),
                  out.stride(0), out.stride(1), _cabi.ptr(lse),
                  lse.stride(0) if lse is not None else 0, _cabi.ptr(scratch),
                  _scratch(scratch), R, prefix_lens.shape[0], int(n_kv), int(G),
                  q.shape[2], k.shape[1], float(scale), _cabi.ptr(status))


def attention_scratch_floats(n_rows: int, n_heads: int, head_dim: int = 128,
                             parts: int = 2) -> int:
    """fp32 elements that ``parts`` partial results of ``n_rows`` query tokens take
    (a maximum, a sum and ``head_dim`` values per head).  Shared-prefix decode needs
    two, and uses up to one per 1 / (KV heads) of the device's SMs and one more."""
    return int(n_rows) * int(n_heads) * (int(head_dim) + 2) * int(parts)
