"""Limits and workspace sizes of the prompt and prefix calls (CPU only: the pointers are never
followed)."""

import pytest

from interattn_amd import _native as N
from tests.test_prompt_refusals import DECODE, prefix_call, refused, struct


@pytest.mark.parametrize("kw", [dict(shape=dict(batch=32769)), dict(shape=dict(batch=1 << 19)), dict(groups=32769),
                                dict(shape=dict(batch=40000, n_q_heads=1, n_kv_heads=1, q_batch_stride=128), groups=0)])
def test_prefix_batches_whose_plan_would_hold_the_device_are_refused(kw):
    refused(prefix_call(**kw), N.IA_ERR_UNSUPPORTED, "batch too large")
    size = N.lib().ia_shared_prefix_workspace_size
    assert size(struct(N.DecodeShape, DECODE, **kw.get("shape", {})), N.IA_BF16, kw.get("groups", 1)) == 0
    assert size(struct(N.DecodeShape, DECODE, batch=32768), N.IA_BF16, 32768) > 0
