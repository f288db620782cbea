"""Prompt rows into pages: the pool, whole, and the lengths equal the rows written one by one."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
CASES = [
    # new, past, hkv, d, page, kv, fused
    ([1], [0], 1, 64, 16, "bf16", False),
    ([37], [100], 8, 128, 16, "bf16", True),
    ([0, 5, 0, 16, 1], [3, 15, 0, 16, 47], 2, 128, 16, "bf16", True),
    ([33, 100], [1, 31], 3, 64, 32, "f32", True),
    ([7, 300], [9, 250], 5, 128, 48, "f32", False),
    ([1000, 1, 777], [0, 5, 64], 8, 128, 16, "bf16", True),
    ([40000], [16], 2, 64, 64, "bf16", False),
]


@pytest.mark.parametrize("c", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("layout", ["split", "paired"])
def test_rows_and_lengths(c, layout, device):
    new, past, hkv, d, page, kv, fused = c
    announce(f"prompt append {c} {layout}")
    gen = torch.Generator(device=device)
    gen.manual_seed(d)
    need = [-(-(a + b) // page) for a, b in zip(new, past)]
    n_pages = sum(need) + 3
    buf = torch.randn((n_pages, hkv, 2, page, d), device=device, generator=gen).to(DT[kv])
    pk, pv = buf[:, :, 0], buf[:, :, 1]
    if layout == "split":
        pk, pv = pk.contiguous(), pv.contiguous()
    table = torch.full((len(new), max(need) + 1), -1, device=device, dtype=torch.int32)
    perm, off = torch.randperm(n_pages, device=device, generator=gen).to(torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = perm[off:off + n]
        off += n
    total = sum(new)
    rows = torch.randn((total + 2, 2 * hkv + 3, d), device=device, generator=gen).to(DT[kv])
    k, v = rows[:, 1:1 + hkv], rows[:, 2 + hkv:2 + 2 * hkv]
    if not fused:
        k, v = k.contiguous(), v.contiguous()
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], device=device, dtype=torch.int32)
    seq = torch.tensor(past, device=device, dtype=torch.int32)
    want_k, want_v, at = pk.clone(), pv.clone(), 0
    for b, n in enumerate(new):
        pos = torch.arange(past[b], past[b] + n, device=device)
        want_k[table[b].long()[pos // page], :, pos % page] = k[at:at + n]
        want_v[table[b].long()[pos // page], :, pos % page] = v[at:at + n]
        at += n
    got = ia.append_prompt_kv(pk, pv, table, seq, k, v, cu)
    torch.cuda.synchronize()
    assert got.tolist() == [a + b for a, b in zip(new, past)] and seq.tolist() == past
    assert torch.equal(pk, want_k) and torch.equal(pv, want_v)


def test_unmapped_pages_end_the_length(device):
    announce("prompt append unmapped")
    hkv, d, page = 2, 64, 16
    pk, pv = (torch.zeros((12, hkv, page, d), device=device) for _ in range(2))
    table = torch.tensor([[0, 1, -1, 3], [4, 99, 5, 6], [7, 8, 9, 10], [-1, 11, -1, -1], [2, -1, -1, -1]],
                         device=device, dtype=torch.int32)
    # row 0: page 2 missing; row 1: page 1 does not exist; row 2: runs past its table row;
    # row 3: its first page is missing; row 4: a negative length takes nothing
    past, new = [10, 0, 50, 5, -1], [40, 60, 20, 20, 3]
    cu = torch.tensor([sum(new[:i]) for i in range(6)], device=device, dtype=torch.int32)
    k = torch.randn((sum(new), hkv, d), device=device)
    out = torch.full((5,), -9, device=device, dtype=torch.int32)
    want = pk.clone()
    at = 0
    for b, n in enumerate(new):
        for i in range(n):
            pos = past[b] + i
            pg = int(table[b, pos // page]) if 0 <= pos < 64 and past[b] >= 0 else -1
            if 0 <= pg < 12:
                want[pg, :, pos % page] = k[at + i]
        at += n
    got = ia.append_prompt_kv(pk, pv, table, torch.tensor(past, device=device, dtype=torch.int32), k, k, cu,
                              new_seq_lens=out)
    torch.cuda.synchronize()
    assert got is out and out.tolist() == [32, 16, 64, 5, -1]
    assert torch.equal(pk, want) and torch.equal(pv, want)
