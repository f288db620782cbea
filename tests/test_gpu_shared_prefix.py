"""Shared-prefix decode against float64 attention of every sequence's whole row, with the
bars of the prompt attention tests (the same products and roundings; the merge of partials
is float32)."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_attention import DT, check, gather, paged, reference

pytestmark = pytest.mark.gpu


def forked(device, members, shared, tails, hkv, d, page, kv, layout, seed):
    """A pool whose tables share each group's whole prefix pages; a prefix's last, partial
    page is repeated in every member's own page."""
    lens = [n + t for n, t in zip([n for m, n in zip(members, shared) for _ in range(m)], tails)]
    pk, pv, scales, table = paged(device, lens, hkv, d, page, kv, layout, seed)
    b = 0
    for m, n in zip(members, shared):
        for i in range(b + 1, b + m):
            table[i, :n // page] = table[b, :n // page]
            if n % page:
                src, dst = int(table[b, n // page]), int(table[i, n // page])
                for pool in (pk, pv):
                    pool.view(torch.uint8)[dst, :, :n % page] = pool.view(torch.uint8)[src, :, :n % page].clone()
                for s in scales or ():
                    s[dst] = s[src]
        b += m
    return pk, pv, scales, table, lens


CASES = [
    # members, shared, tails, hq, hkv, d, page, kv, layout
    ([2], [16], [0, 1], 4, 1, 128, 16, "bf16", "split"),
    ([3], [5], [0, 3, 40], 4, 2, 64, 16, "bf16", "split"),
    ([4, 1, 2], [333, 70, 1000], [1, 0, 17, 200, 9, 63, 65], 8, 2, 128, 16, "bf16", "paired"),
    ([33], [2000], list(range(33)), 32, 8, 128, 16, "bf16", "split"),
    ([10], [4097], [7] * 10, 8, 1, 64, 32, "bf16", "split"),
    ([5, 3], [513, 64], [0] * 8, 6, 2, 128, 48, "bf16", "split"),
    ([1, 1], [100, 0], [5, 6], 8, 2, 128, 16, "bf16", "split"),
    ([3, 4], [200, 1500], [2, 90, 0, 33, 7, 1, 300], 8, 2, 128, 16, "fp8", "paired"),
    ([40], [700], [3] * 40, 4, 1, 64, 32, "fp8", "split"),
    ([3, 2], [100, 900], [1, 2, 30, 0, 64], 8, 4, 128, 16, "f32", "split"),
    ([20], [600], [5] * 20, 16, 2, 64, 16, "f32", "paired"),
]


@pytest.mark.parametrize("c", CASES, ids=[f"{c[7]}-{c[5]}-{c[3]}x{c[4]}-{i}" for i, c in enumerate(CASES)])
def test_against_whole_rows(c, device):
    members, shared, tails, hq, hkv, d, page, kv, layout = c
    announce(f"shared prefix {c}")
    pk, pv, scales, table, lens = forked(device, members, shared, tails, hkv, d, page, kv, layout, d + len(tails))
    gen = torch.Generator(device=device)
    gen.manual_seed(1)
    q = torch.randn((len(lens), hq, d), device=device, generator=gen).to(DT["f32" if kv == "f32" else "bf16"])
    seq = torch.tensor(lens, device=device, dtype=torch.int32)
    starts = torch.tensor([sum(members[:i]) for i in range(len(members) + 1)], device=device, dtype=torch.int32)
    sh = torch.tensor(shared, device=device, dtype=torch.int32)
    ws = {}
    out = ia.shared_prefix_decode(q, pk, pv, table, seq, starts, sh, scales=scales, workspace=ws)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        k = gather(pk, scales and scales[0], table[b], n)
        v = gather(pv, scales and scales[1], table[b], n)
        want, mag = reference(q[b:b + 1], k, v, n - 1, d ** -0.5)
        check(out[b:b + 1], want, mag, kv, n, (c, b))
    # again in the same workspace, without the groups: every sequence by itself
    alone = ia.shared_prefix_decode(q, pk, pv, table, seq, starts[:1], sh[:0], scales=scales, workspace=ws,
                                    out=torch.empty_like(out))
    for b, n in enumerate(lens):
        k = gather(pk, scales and scales[0], table[b], n)
        v = gather(pv, scales and scales[1], table[b], n)
        want, mag = reference(q[b:b + 1], k, v, n - 1, d ** -0.5)
        check(alone[b:b + 1], want, mag, kv, n, ("alone", c, b))


def test_sequences_of_no_group_and_short_members(device):
    """Sequences before, between and behind the groups; a member shorter than its prefix; a
    first sequence shorter than the stated prefix; empty sequences; an empty group."""
    announce("shared prefix odd groups")
    hkv, hq, d, page = 2, 8, 128, 16
    lens = [50, 300, 120, 310, 0, 90, 40, 41, 77]
    pk, pv, _, table = paged(device, lens, hkv, d, page, "bf16", "split", 3)
    # sequences 1..3 share 200 tokens, 3 is longer, 2 has only 120; 6..7 claim 64 but have 40
    for i in (2, 3):
        whole = min(lens[i], 200) // page
        table[i, :whole] = table[1, :whole]
    for pool in (pk, pv):
        pool[int(table[3, 12]), :, :8] = pool[int(table[1, 12]), :, :8].clone()
        pool[int(table[2, 7]), :, :8] = pool[int(table[1, 7]), :, :8].clone()
        for pg in range(3):
            pool[int(table[7, pg])] = pool[int(table[6, pg])].clone()
    q = torch.randn((len(lens), hq, d), device=device).to(torch.bfloat16)
    seq = torch.tensor(lens, device=device, dtype=torch.int32)
    starts = torch.tensor([1, 4, 4, 6, 8], device=device, dtype=torch.int32)
    shared = torch.tensor([200, 5, 0, 64], device=device, dtype=torch.int32)
    out = ia.shared_prefix_decode(q, pk, pv, table, seq, starts, shared, workspace={})
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        want, mag = reference(q[b:b + 1], gather(pk, None, table[b], n), gather(pv, None, table[b], n), n - 1, d ** -0.5)
        check(out[b:b + 1], want, mag, "bf16", n, b)
    assert bool((out[4] == 0).all())
