"""MI355X-native (gfx950) condition-block sparse decode attention.

The compute path is the HIP library ``libinterattn_amd.so`` (C ABI in
``include/interattn_amd.h``); this package is its torch-facing host side.
"""

from ._native import NativeLibraryMissing, NativeError  # noqa: F401
from .beam import beam_select  # noqa: F401
from .ops import (  # noqa: F401
    append_kv,
    build_block_summaries,
    paged_decode,
    paged_kv,
    select_blocks_topk,
    sequence_scales,
    set_wait_limit,
    sparse_paged_decode,
    sparse_topk_decode,
    update_block_summaries,
    wait_fallbacks,
    workspace_tensor,
)
from .pages import (  # noqa: F401
    compact_pages,
    copy_pages,
    fork_sequences,
    free_sequences,
    reorder_sequences,
    reserve_pages,
)
from .prompt import (  # noqa: F401
    append_prompt_kv,
    paged_prompt_attention,
    prompt_attention,
    read_kv,
    shared_prefix_decode,
)
from .rotary import RotaryPlan, apply_rotary, rotary_append_kv, rotary_frequencies, rotary_plan  # noqa: F401

__version__ = "0.1.0"
