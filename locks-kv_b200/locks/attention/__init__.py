"""Stage B -- sparse paged attention over the selected pages, and the serving step
around it: slots of new tokens, head norms with rotation into the cache, attention
with a sliding window, decode over a shared prefix."""
from __future__ import annotations

from .append_plan import append_plan  # noqa: F401
from .decode import (DenseDecodeBuffers, PinnedHostVSource,  # noqa: F401
                     ResidentVSource, VSource,
                     dense_paged_decode, ensure_stage_b_buffers,
                     sparse_paged_decode_batched, sparse_paged_decode_fused)
from .kv_write import (kv_append_desc, norm_rope_and_cache,  # noqa: F401
                       rope_and_cache)
from .merge import merge_splits  # noqa: F401
from .paged import (attention_scratch_floats,  # noqa: F401
                    shared_prefix_paged_decode, window_paged_attention)

__all__ = ["sparse_paged_decode_batched", "sparse_paged_decode_fused",
           "dense_paged_decode", "DenseDecodeBuffers", "ResidentVSource",
           "PinnedHostVSource",
           "VSource", "ensure_stage_b_buffers", "merge_splits", "rope_and_cache",
           "kv_append_desc", "append_plan", "norm_rope_and_cache",
           "window_paged_attention", "shared_prefix_paged_decode",
           "attention_scratch_floats"]
