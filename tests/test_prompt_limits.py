"""Limits and workspace sizes of the prompt and prefix calls (CPU only: the pointers are never
followed)."""

import random

import pytest

from interattn_amd import _native as N
from tests.test_prompt_refusals import BIG, DECODE, KV, P, SHAPE, STATE, append_call, prefix_call, refused, struct


@pytest.mark.parametrize("kw", [dict(shape=dict(batch=32769)), dict(shape=dict(batch=1 << 19)), dict(groups=32769),
                                dict(shape=dict(batch=40000, n_q_heads=1, n_kv_heads=1, q_batch_stride=128), groups=0)])
def test_prefix_batches_whose_plan_would_hold_the_device_are_refused(kw):
    refused(prefix_call(**kw), N.IA_ERR_UNSUPPORTED, "batch too large")
    size = N.lib().ia_shared_prefix_workspace_size
    assert size(struct(N.DecodeShape, DECODE, **kw.get("shape", {})), N.IA_BF16, kw.get("groups", 1)) == 0
    assert size(struct(N.DecodeShape, DECODE, batch=32768), N.IA_BF16, 32768) > 0


def test_prefix_scratch_is_what_its_partials_need():
    """Two partial rows for each query row, and what the cuts add: at most 64 items of 128
    rows per kv head (512 workgroups of 8 heads)."""
    size = lambda batch, groups: N.lib().ia_shared_prefix_workspace_size(  # noqa: E731
        struct(N.DecodeShape, DECODE, batch=batch, n_q_heads=32, n_kv_heads=8), N.IA_BF16, groups)
    row = 8 * 130 * 4  # eight heads' (acc, m, l)
    for batch, groups in ((1, 0), (32, 1), (64, 8), (512, 256), (4096, 4096)):
        rows = 2 * 4 * batch + 64 * 128
        plan = 16 * (batch + batch // 32 + groups)
        assert size(batch, groups) <= rows * row + plan + 4 * 256, (batch, groups)
    # more of either never needs less
    assert size(40, 3) <= size(64, 64) <= size(65, 64) and size(64, 64) <= size(64, 65)


def test_arrays_without_entries_may_be_null():
    lib = N.lib()
    none = struct(N.DecodeShape, DECODE, batch=0)
    assert lib.ia_shared_prefix_decode(none, None, struct(N.PagedKV, KV), None, None, None, 0, 0.1, None, N.IA_BF16,
                                       None, 0, None) == N.IA_OK
    assert append_call(cu=None, seq=None, new=None, n_seq=0) == N.IA_OK
    for kw in (dict(rows=0, block_table=None, seq_lens=None), dict(rows=0, block_table=None, seq_lens=None, n_pages=0,
                                                                   refs=None)):
        assert lib.ia_reserve_pages(struct(N.PageState, STATE, **kw), None, None, None, 0, None) == N.IA_OK
        assert lib.ia_free_sequences(struct(N.PageState, STATE, **kw), None, 0, None) == N.IA_OK
    for kw in (dict(block_table=None), dict(seq_lens=None), dict(refs=None)):
        refused(lib.ia_reserve_pages(struct(N.PageState, STATE, **kw), P, P, P, BIG, None), N.IA_ERR_INVALID, "null")


def test_a_packed_call_is_never_cut_without_workspace():
    """Callers size the workspace for n_tokens keys; the call cuts for the mean length."""
    rng = random.Random(0)
    size = N.lib().ia_prompt_attention_workspace_size
    cut = 0
    for _ in range(20000):
        hkv, g = rng.choice([1, 2, 3, 4, 8, 32]), rng.choice([1, 2, 3, 4, 6, 8, 16, 32, 40, 64])
        n_seq, tokens = int(2 ** rng.uniform(0, 9)), int(2 ** rng.uniform(0, 17))
        shape = struct(N.PromptShape, SHAPE, n_seq=n_seq, n_tokens=tokens, n_q_heads=hkv * g, n_kv_heads=hkv)
        kv = rng.choice([N.IA_BF16, N.IA_F32])
        mean = size(shape, kv, -(-tokens // n_seq))
        cut += mean > 0
        assert mean == 0 or size(shape, kv, tokens) == mean, (hkv, g, n_seq, tokens, kv)
    assert cut > 100
