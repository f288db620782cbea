"""Batches, tables and lists without entries (an empty tensor has no address)."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce
from tests.test_gpu_prompt_edges import i32

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 4, 2, 64, 16


def pools(device, n_pages=6):
    return tuple(torch.randn((n_pages, HKV, PAGE, D), device=device).to(torch.bfloat16) for _ in range(2))


def rows(device, n, heads):
    return torch.randn((n, heads, D), device=device).to(torch.bfloat16)


def table(device, *shape):
    return torch.full(shape, -1, device=device, dtype=torch.int32)


def test_attention_of_nothing(device):
    announce("empty attention")
    pk, pv = pools(device)
    none, one = i32(device, []), i32(device, [0])
    q = rows(device, 0, HQ)
    assert ia.prompt_attention(q, rows(device, 0, HKV), rows(device, 0, HKV), one).shape == q.shape
    assert ia.prompt_attention(q, rows(device, 0, HKV), rows(device, 0, HKV), i32(device, [0, 0, 0])).shape == q.shape
    assert ia.paged_prompt_attention(q, pk, pv, table(device, 0, 3), none, one).shape == q.shape
    assert ia.shared_prefix_decode(q, pk, pv, table(device, 0, 3), none, one, none).shape == q.shape
    assert ia.shared_prefix_decode(q, pk, pv, table(device, 0, 3), none, i32(device, [0, 0]), one).shape == q.shape
    # rows of no sequence
    out = torch.full((5, HQ, D), 3.0, device=device, dtype=torch.bfloat16)
    ia.prompt_attention(rows(device, 5, HQ), rows(device, 5, HKV), rows(device, 5, HKV), one, out=out)
    torch.cuda.synchronize()
    assert bool((out == 3.0).all())


def test_append_of_nothing(device):
    announce("empty append")
    pk, pv = pools(device)
    k0, v0 = pk.clone(), pv.clone()
    for n in (0, 4):
        new = rows(device, n, HKV)
        assert ia.append_prompt_kv(pk, pv, table(device, 0, 3), i32(device, []), new, new, i32(device, [0])).numel() == 0
    new = rows(device, 0, HKV)
    lens = ia.append_prompt_kv(pk, pv, table(device, 2, 3), i32(device, [7, 0]), new, new, i32(device, [0, 0, 0]))
    torch.cuda.synchronize()
    assert lens.tolist() == [7, 0] and torch.equal(pk, k0) and torch.equal(pv, v0)


def test_tables_without_columns_hold_no_token(device):
    """A table of no columns is not the identity table that None stands for."""
    announce("tables without columns")
    pk, pv = pools(device)
    k0 = pk.clone()
    t, lens = table(device, 2, 0), i32(device, [20, 0])
    out = ia.paged_prompt_attention(rows(device, 2, HQ), pk, pv, t, lens, i32(device, [0, 1, 2]))
    one = ia.shared_prefix_decode(rows(device, 2, HQ), pk, pv, t, lens, i32(device, [0, 2]), i32(device, [16]))
    new = rows(device, 3, HKV)
    after = ia.append_prompt_kv(pk, pv, t, i32(device, [0, 0]), new, new, i32(device, [0, 2, 3]))
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((one == 0).all())
    assert after.tolist() == [0, 0] and torch.equal(pk, k0)


def test_pages_of_tables_without_rows(device):
    announce("empty page states")
    pk, pv = pools(device)
    k0 = pk.clone()
    t, none = table(device, 0, 3), i32(device, [])
    refs = i32(device, [0, 0, 1, 0, 0, 2])
    assert ia.reserve_pages(t, none, refs, none, page_size=PAGE).numel() == 0
    assert ia.fork_sequences([pk, pv], t, none, refs, none, none, page_size=PAGE).numel() == 0
    assert ia.fork_sequences([pk, pv], t, none, refs, i32(device, [0]), i32(device, [1]), page_size=PAGE).tolist() == [0]
    ia.free_sequences(t, none, refs, i32(device, [0]))
    ia.free_sequences(t, none, refs, none)
    ia.copy_pages([pk, pv], none, none)
    torch.cuda.synchronize()
    assert refs.tolist() == [0, 0, 1, 0, 0, 2] and torch.equal(pk, k0)
    # pages held by nobody's row are still held
    assert ia.compact_pages([pk, pv], t, refs).tolist() == [2]
    assert refs.tolist() == [1, 2, 0, 0, 0, 0] and torch.equal(pk[:2], k0[[2, 5]])
    # rows without columns, pools without pages
    assert ia.reserve_pages(table(device, 2, 0), i32(device, [0, 0]), refs, i32(device, [0, 1]),
                            page_size=PAGE).tolist() == [1, 0]
    assert ia.reserve_pages(table(device, 2, 3), i32(device, [0, 0]), none, i32(device, [0, 1]),
                            page_size=PAGE).tolist() == [1, 0]
    assert ia.compact_pages([], table(device, 2, 3), none).tolist() == [0]
