"""The tensors of a page call may come from any iterable: a generator, a chain, a map, a view."""

import itertools

import pytest
import torch

import interattn_amd as ia
from interattn_amd import pages
from tests._util import announce

FORMS = {
    "list": list,
    "generator": lambda ts: (t for t in ts),
    "chain": lambda ts: itertools.chain(ts[::2], ts[1::2]),
    "map": lambda ts: map(lambda t: t, ts),
    "values": lambda ts: dict(enumerate(ts)).values(),
}


@pytest.mark.parametrize("form", FORMS)
def test_every_tensor_is_described(form):
    refs = torch.zeros(6, dtype=torch.int32)
    ts = [torch.zeros((6, 2, 16, 64)), torch.zeros((6, 2, 16, 64)), torch.zeros((6, 2)), torch.zeros((6, 3, 16))[:, 1]]
    order = list(FORMS[form](ts))
    desc, n, n_pages = pages._page_tensors(FORMS[form](ts), None, refs)
    assert n == len(ts) and n_pages == 6
    assert [d.data for d in desc] == [t.data_ptr() for t in order]
    assert [d.run_bytes for d in desc] == [{4: 2 * 16 * 64 * 4, 2: t.shape[1] * 4}[t.dim()] for t in order]
    assert pages._page_tensors(FORMS[form]([]), 6, refs) == (None, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_page_calls_take_them(device, form):
    """Each of the four calls moves the pages of every tensor, as with a list."""
    announce(f"page tensors from a {form}")
    g = torch.Generator(device=device)
    g.manual_seed(2)
    start = [torch.randn((8, 2, 16, 64), device=device, generator=g) for _ in range(3)]
    start.append(torch.rand((8, 2), device=device, generator=g))

    def ints(*x):
        return torch.tensor(x, device=device, dtype=torch.int32)

    def copy(ts, table, lens, refs):
        ia.copy_pages(ts, ints(0, 5), ints(6, 7))

    def fork(ts, table, lens, refs):
        assert ia.fork_sequences(ts, table, lens, refs, ints(0), ints(2), page_size=16).tolist() == [1]

    def reorder(ts, table, lens, refs):
        assert ia.reorder_sequences(ts, table, lens, refs, ints(1, 1, 0), page_size=16).tolist() == [1] * 3

    def compact(ts, table, lens, refs):
        assert ia.compact_pages(ts, table, refs).tolist() == [4]

    for call in (copy, fork, reorder, compact):
        got = []
        for make in (list, FORMS[form]):
            ts = [t.clone() for t in start]
            state = (torch.tensor([[5, 1, -1], [7, 3, -1], [-1, -1, -1]], device=device, dtype=torch.int32),
                     ints(20, 30, 0), ints(0, 1, 0, 1, 0, 1, 0, 1))
            call(make(ts), *state)
            torch.cuda.synchronize()
            got.append([*ts, *state])
        assert all(torch.equal(a, b) for a, b in zip(*got))
        assert not all(torch.equal(a, b) for a, b in zip(got[0], start))
