"""Stage B: sparse paged attention over the selected pages, and what stands around it:
the cache write of a projection, window, prompt and shared-prefix attention."""
from .decode import (ResidentVSource, decode_dense, decode_merge, decode_splitk, decode_splitk_tier,  # noqa: F401
                     ensure_stage_b_buffers, sparse_paged_decode_batched)
from .mla_decode import mla_decode, mla_decode_dense  # noqa: F401
from .qkv import qk_norm_rope_write  # noqa: F401
from .window import attn_workspace, prefix_decode, window_decode, window_prefill  # noqa: F401
