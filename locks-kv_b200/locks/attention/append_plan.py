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
    refused as a whole: slots -1, nothing else changed for it, ``status`` 3; behind
    one refused for want of blocks only requests that need none are served."""
    dev = _cabi.one_device(seq_lens, n_new, block_table, free_blocks, taken,
                           slot_mapping, positions, cu_tokens, lens_out, taken_out,
                           status)
    i32, i64 = torch.int32, torch.int64
    for t in (seq_lens, n_new, free_blocks, taken, cu_tokens, lens_out, taken_out):
        assert t.dtype is i32 and t.is_contiguous(), \
            "lengths, counts and the free list are contiguous int32"
    assert slot_mapping.dtype is i64 and slot_mapping.is_contiguous()
    assert positions.dtype is i64 and positions.is_contiguous()
    assert status is None or status.dtype is i32, "status is int32"
    R, cap = seq_lens.numel(), slot_mapping.numel()
    rows, width = block_table.shape
    stride = block_table.stride()
    assert block_table.dtype is i32 and stride[1] == 1
    assert n_new.numel() == lens_out.numel() == rows == R
    assert cu_tokens.numel() == R + 1 and positions.numel() == cap
    assert taken.numel() == taken_out.numel() == 1
    if R == 0:
        cu_tokens.zero_()
        slot_mapping.fill_(-1)
        positions.zero_()
        if taken_out.data_ptr() != taken.data_ptr():
            taken_out.copy_(taken)
        return
    _cabi.call_on(dev, "locks_append_plan", seq_lens.data_ptr(), n_new.data_ptr(),
                  block_table.data_ptr(), width if R == 1 else stride[0], width,
                  free_blocks.data_ptr(), free_blocks.numel(), taken.data_ptr(),
                  slot_mapping.data_ptr(), positions.data_ptr(), cu_tokens.data_ptr(),
                  lens_out.data_ptr(), taken_out.data_ptr(), R, cap, page,
                  _cabi.addr(status))
