"""Where an append writes the lengths after it: not over lengths or row starts that other
workgroups of the call still read."""

import pytest

from interattn_amd import _native as N

P = 1 << 32  # an aligned address that nothing follows
SEQS, D = 5, 128
CU, LENS, NEW = P, P + 4096, P + 8192


def refused(rc, what):
    msg = N.lib().ia_last_error().decode()
    assert rc == N.IA_ERR_INVALID and "new_seq_lens" in msg and what in msg, (rc, msg)


def calls(cu, lens, new, single):
    kv = N.PagedKV(P + (1 << 30), P + (1 << 31), N.IA_BF16, 16, 9, 16 * D, 16 * D, D, 16 * D, 16 * D, D, P - 4096, 4, 4)
    rows = N.PackedKV(P + (1 << 28), P + (1 << 29), N.IA_BF16, D, 0, D, 0)
    lib, tokens = N.lib(), SEQS if single else 40
    yield lib.ia_rotary_append_kv(None, None, rows, kv, None if single else cu, lens, new, None, SEQS, tokens, 1, D, None)
    if not single:
        yield lib.ia_append_prompt_kv(kv, rows, cu, lens, new, SEQS, tokens, 1, D, None)


@pytest.mark.parametrize("new", [CU, CU + 4, CU - 4 * (SEQS - 1), CU + 4 * SEQS])
def test_over_the_row_starts(new):
    for rc in calls(CU, LENS, new, False):
        refused(rc, "cu_seqlens")


@pytest.mark.parametrize("single", [False, True])
@pytest.mark.parametrize("apart", [4, -4, 4 * (SEQS - 1), -4 * (SEQS - 1)])
def test_partly_over_the_lengths(apart, single):
    for rc in calls(CU, LENS, LENS + apart, single):
        refused(rc, "seq_lens")
