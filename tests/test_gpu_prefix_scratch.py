"""The shared-prefix call's scratch: few buffers for a server whose batch changes, none
replaced, and groups that do not fit the plan's assumptions stay inside it."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import check, gather, paged, reference
from tests.test_gpu_prompt_edges import i32

pytestmark = pytest.mark.gpu


def test_one_buffer_serves_batches_that_change(device):
    announce("prefix scratch, changing batch")
    hkv, hq, d, page = 8, 32, 128, 16
    lens = [20 + i % 7 for i in range(80)]
    pk, pv, _, table = paged(device, lens, hkv, d, page, "bf16", "split", 2)
    q = torch.randn((80, hq, d), device=device).to(torch.bfloat16)
    ws, seen = {}, {}
    for b in (1, 2, 3, 7, 13, 24, 48, 64, 80):
        for groups in (1, 2, 5):
            starts = [min(i, b) for i in range(groups + 1)]  # (groups of one)
            out = ia.shared_prefix_decode(q[:b], pk, pv, table[:b], i32(device, lens[:b]), i32(device, starts),
                                          i32(device, [16] * groups), workspace=ws)
            for key, t in ws.items():
                if t.dtype == torch.uint8:
                    assert seen.setdefault(key, t.data_ptr()) == t.data_ptr(), "a buffer was replaced"
    torch.cuda.synchronize()
    scratch = [t.numel() for t in ws.values() if t.dtype == torch.uint8]
    assert len(scratch) == 2 and sum(scratch) < 100 << 20, scratch
    for i in (0, 40, 79):
        n = lens[i]
        want, mag = reference(q[i:i + 1], gather(pk, None, table[i], n), gather(pv, None, table[i], n), n - 1, d ** -0.5)
        check(out[i:i + 1], want, mag, "bf16", n, i)


def test_starts_that_put_sequences_in_many_groups_stay_inside(device):
    """group_starts must not decrease; these put all 32 sequences into each of 300 groups, more
    partial rows than the scratch has.  What follows the scratch is left alone."""
    announce("prefix scratch, overlapping groups")
    hkv, hq, d, page, b, groups = 1, 64, 64, 16, 32, 300
    pk, pv, _, table = paged(device, [40] * b, hkv, d, page, "bf16", "split", 3)
    q = torch.randn((b, hq, d), device=device).to(torch.bfloat16)
    starts = i32(device, [0 if i % 2 == 0 else b for i in range(groups + 1)])
    ws = {}
    args = (q, pk, pv, table, i32(device, [40] * b), starts, i32(device, [32] * groups))
    ia.shared_prefix_decode(*args, workspace=ws)
    (key, t), = [(k, t) for k, t in ws.items() if t.dtype == torch.uint8]
    held = torch.full((t.numel() + (1 << 22) + 256,), 77, device=device, dtype=torch.uint8)
    off = -held.data_ptr() % 256
    ws[key] = held[off:off + t.numel()]
    ia.shared_prefix_decode(*args, workspace=ws)
    torch.cuda.synchronize()
    assert bool((held[off + t.numel():] == 77).all()) and bool((held[:off] == 77).all())
