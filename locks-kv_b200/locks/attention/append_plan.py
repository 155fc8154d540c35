"""Step bookkeeping on the device (host wrapper of ``locks_append_plan``).

``append_advance`` (selection) is the one-token-per-request form for a captured
decode loop whose blocks are in the table already; this one takes any number of
new tokens per request and hands out blocks from a free list.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi


def append_plan(seq_lens: torch.Tensor, n_new: torch.Tensor,
                block_table: torch.Tensor, free_blocks: torch.Tensor,
                taken: torch.Tensor, *, slot_mapping: torch.Tensor,
                positions: torch.Tensor, cu_tokens: torch.Tensor,
                lens_out: torch.Tensor, taken_out: torch.Tensor, page: int = 16,
                status: Optional[torch.Tensor] = None) -> None:
    """seq_lens, n_new: int32 (R,), tokens cached before the step and new ones.
    block_table: int32 (R, W), updated in place.  free_blocks: int32 (F,), of which
    the first ``taken`` (int32, one element) are handed out already.

    Written: ``slot_mapping`` / ``positions`` int64 (T,) in the token layout of
    ``cu_tokens`` int32 (R + 1,), -1 / 0 behind the last token; ``lens_out`` int32
    (R,) and ``taken_out`` int32, one element (may be ``seq_lens`` and ``taken``
    themselves).  A request that does not fit its table row, the free list or T is
    refused as a whole: slots -1, nothing else changed for it, ``status`` 3."""
    dev = _cabi.one_device(seq_lens, n_new, block_table, free_blocks, taken,
                           slot_mapping, positions, cu_tokens, lens_out, taken_out,
                           status)
    R = seq_lens.shape[0]
    for t in (seq_lens, n_new, free_blocks, taken, cu_tokens, lens_out, taken_out):
        assert t.dtype == torch.int32 and t.is_contiguous(), \
            "lengths, counts and the free list are contiguous int32"
    assert slot_mapping.dtype == positions.dtype == torch.int64
    assert slot_mapping.is_contiguous() and positions.is_contiguous()
    assert block_table.dtype == torch.int32 and block_table.stride(1) == 1
    assert n_new.shape[0] == lens_out.shape[0] == block_table.shape[0] == R
    assert cu_tokens.shape[0] == R + 1
    assert positions.shape == slot_mapping.shape
    assert taken.numel() == taken_out.numel() == 1
    if R == 0:
        cu_tokens.zero_()
        slot_mapping.fill_(-1)
        positions.zero_()
        if taken_out.data_ptr() != taken.data_ptr():
            taken_out.copy_(taken)
        return
    _cabi.call_on(dev, "locks_append_plan", _cabi.ptr(seq_lens), _cabi.ptr(n_new),
                  _cabi.ptr(block_table), max(block_table.stride(0), block_table.shape[1])
                  if R == 1 else block_table.stride(0), block_table.shape[1],
                  _cabi.ptr(free_blocks), free_blocks.shape[0], _cabi.ptr(taken),
                  _cabi.ptr(slot_mapping), _cabi.ptr(positions), _cabi.ptr(cu_tokens),
                  _cabi.ptr(lens_out), _cabi.ptr(taken_out), R, slot_mapping.shape[0],
                  int(page), _cabi.ptr(status))
