"""Rows that follow their parents, against the oracle, exactly: tables, lengths, counts, pages."""

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import beam as B
from tests._util import announce

pytestmark = pytest.mark.gpu


def make(device, seed, rows, cols, page, lens, n_pages, share=0, reserve=0, layers=2, fp8=False):
    """Rows of the given lengths; ``share`` of the neighbours' leading pages are common, ``reserve``
    pages are mapped past the length."""
    rng = np.random.default_rng(seed)
    free = list(rng.permutation(n_pages))
    table = np.full((rows, cols), -1, np.int32)
    for i, n in enumerate(lens):
        need = min(-(-n // page) + reserve, cols)
        for c in range(need):
            if c < share and i % 4 and c < lens[i] // page and c < lens[i - 1] // page:
                table[i, c] = table[i - 1, c]
            else:
                table[i, c] = free.pop()
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    tensors = []
    for layer in range(layers):
        kv = torch.randint(0, 256, (n_pages, 2, 2, page, 64), device=device, generator=g).to(torch.uint8)
        if layer % 2:
            tensors += [kv[:, :, 0], kv[:, :, 1]]
        else:
            tensors += [kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous()]
        if fp8:
            tensors += [torch.rand((n_pages, 2), device=device, generator=g) for _ in "kv"]
    dev = [torch.from_numpy(x).to(device) for x in (table, np.array(lens, np.int32), refs)]
    return tensors, dev


def run(device, tensors, state, parents, page, workspace=None):
    table, lens, refs = state
    want = B.reorder(*(x.cpu().numpy() for x in state), np.array(parents), page)
    moved = [t.clone() for t in tensors]
    for src, dst in want[4]:
        for t in moved:
            t[dst] = t[src]
    ok = ia.reorder_sequences(tensors, table, lens, refs, torch.tensor(parents, device=device, dtype=torch.int32),
                              page_size=page, workspace=workspace)
    torch.cuda.synchronize()
    for got, w in zip((table, lens, refs, ok), want[:4]):
        assert np.array_equal(got.cpu().numpy(), w), (got.cpu().numpy(), w)
    for a, b in zip(tensors, moved):
        assert torch.equal(a, b)
    return ok


CASES = [
    ("alone", [37], 3, [0]),
    ("nothing changes", [37, 20, 16], 3, [0, 1, 2]),
    ("swap", [37, 20], 3, [1, 0]),
    ("cycle", [37, 20, 16, 1], 3, [3, 0, 1, 2]),
    ("all of one", [37, 20, 16, 40], 3, [1, 1, 1, 1]),
    ("all of the last", [37, 20, 16, 41], 3, [3, 3, 3, 3]),
    ("whole pages only", [32, 48, 16, 0], 3, [1, 0, 0, 0]),
    ("empty parents", [0, 48, 0, 5], 3, [0, 0, 2, 2]),
    ("ended", [33, 48, 7, 5], 3, [-1, 1, 9, -1]),
    ("ended parent", [33, 48, 7, 5], 3, [-1, 0, 0, 3]),
    ("full rows", [48, 48, 48], 3, [2, 2, 0]),
    ("two families", [37, 20, 33, 40, 21, 22, 23, 24], 3, [1, 1, 0, 0, 7, 4, 4, 4]),
]


@pytest.mark.parametrize("name,lens,cols,parents", CASES, ids=[c[0] for c in CASES])
@pytest.mark.parametrize("share,reserve,fp8", [(0, 0, False), (2, 1, True)])
def test_rows_follow_their_parents(device, name, lens, cols, parents, share, reserve, fp8):
    announce(f"reorder {name} {share} {reserve}")
    tensors, state = make(device, len(lens), len(lens), cols + reserve, 16, lens, 64, share, reserve, fp8=fp8)
    ok = run(device, tensors, state, parents, 16)
    assert bool(ok.all())
    # and again, on what it left
    run(device, tensors, state, parents, 16)


@pytest.mark.parametrize("seed", range(8))
def test_many_steps(device, seed):
    """Random parents over many steps, lengths growing between, on one workspace."""
    announce(f"reorder, steps {seed}")
    rng = np.random.default_rng(seed)
    rows, page, cols = [3, 8, 40, 1, 70, 5, 16, 33][seed], [16, 32, 16, 16, 64, 16, 48, 16][seed], [5, 4, 9, 6, 3, 300, 4, 2][seed]
    n_pages = rows * cols + rows + 3
    lens = rng.integers(1, cols * page // 2 + 1, rows).tolist()
    tensors, state = make(device, seed, rows, cols, page, lens, n_pages, layers=1)
    ws = {}
    for _ in range(6):
        run(device, tensors, state, rng.integers(0, rows, rows).tolist(), page, ws)
        ia.reserve_pages(*state, torch.ones(rows, device=device, dtype=torch.int32), page_size=page)
        room = state[1] < cols * page
        state[1].add_((room & (state[0].gather(1, (state[1] // page).clamp_max(cols - 1).long()[:, None])[:, 0] >= 0)).int())


def test_rows_that_cannot_follow(device):
    """A partly filled page that is not mapped, lengths that do not fit, no page left."""
    announce("reorder, failures")
    lens = [37, 20, 16, 5]
    tensors, state = make(device, 1, 4, 3, 16, lens, 12)
    state[0][0, 2] = -1
    ok = run(device, tensors, state, [0, 0, 2, 3], 16)
    assert ok.tolist() == [1, 0, 1, 1] and state[1].tolist() == [37, 0, 16, 5]
    for bad in (-4, 49, 2 ** 31 - 1):
        tensors, state = make(device, 1, 4, 3, 16, lens, 12)
        state[1][3] = bad
        ok = run(device, tensors, state, [0, 3, 2, 3], 16)
        assert ok.tolist() == [1, 0, 1, 1] and state[1].tolist() == [37, 0, 16, bad]
        run(device, tensors, state, [3, 1, 2, 2], 16)  # an heir takes it as it is
    # seven pages, all held; dropping rows 2 and 3 frees two, three copies are asked for
    tensors, state = make(device, 1, 5, 3, 16, [37, 20, 16, 5, 2], 8)
    ok = run(device, tensors, state, [0, 1, 0, 1, 0], 16)
    assert ok.tolist() == [1, 1, 1, 1, 1]
    tensors, state = make(device, 1, 4, 3, 16, [37, 20, 16, 32], 8)
    state[2][state[2] == 0] = 1  # (held elsewhere)
    ok = run(device, tensors, state, [0, 0, 0, 3], 16)
    assert ok.tolist() == [1, 1, 1, 1]
    tensors, state = make(device, 1, 3, 3, 16, [48, 37, 37], 9)
    state[2][state[2] == 0] = 1
    ok = run(device, tensors, state, [0, 1, 1], 16)
    assert ok.tolist() == [1, 1, 1]
    tensors, state = make(device, 1, 4, 3, 16, [48, 37, 32, 0], 8)
    state[2][state[2] == 0] = 1
    ok = run(device, tensors, state, [0, 1, 2, 1], 16)
    assert ok.tolist() == [1, 1, 1, 0] and state[1].tolist() == [48, 37, 32, 0]


def test_strided_tables_many_tensors_no_columns(device):
    announce("reorder, layouts")
    tensors, state = make(device, 2, 6, 3, 16, [37, 20, 16, 40, 1, 0], 40, layers=30)
    wide = torch.full((6, 50), 77, device=device, dtype=torch.int32)
    wide[:, 5:8] = state[0]
    state[0] = wide[:, 5:8]
    run(device, tensors, state, [3, 3, 0, 0, 3, 1], 16)
    assert bool((wide[:, :5] == 77).all()) and bool((wide[:, 8:] == 77).all())
    # a table of no columns: only lengths move
    table = torch.zeros((3, 0), device=device, dtype=torch.int32)
    lens, refs = torch.zeros(3, device=device, dtype=torch.int32), torch.zeros(4, device=device, dtype=torch.int32)
    ok = ia.reorder_sequences([], table, lens, refs, torch.tensor([1, 1, -1], device=device, dtype=torch.int32), page_size=16)
    torch.cuda.synchronize()
    assert ok.tolist() == [1, 1, 1] and lens.tolist() == [0, 0, 0]
    ok = ia.reorder_sequences([], table[:0], lens[:0], refs, lens[:0], page_size=16)
    assert ok.shape == (0,)


@pytest.mark.parametrize("rows,cols,longest", [(4, 9001, 144000), (1500, 3, 40), (2, 4097, 65552)])
def test_wide_tables_and_many_rows(device, rows, cols, longest):
    """Tables wider than a workgroup's stretch of columns, more rows than a workgroup's threads."""
    announce(f"reorder, {rows} rows of {cols} pages")
    rng = np.random.default_rng(rows)
    lens = rng.integers(0, longest + 1, rows).tolist()
    lens[0] = longest
    n_pages = sum(-(-n // 16) for n in lens) + rows
    g = torch.Generator(device=device)
    g.manual_seed(rows)
    table, free = np.full((rows, cols), -1, np.int32), rng.permutation(n_pages)
    for i, n in enumerate(lens):
        need = -(-n // 16)
        table[i, :need], free = free[:need], free[need:]
    refs = np.bincount(table[table >= 0], minlength=n_pages).astype(np.int32)
    tensors = [torch.randint(0, 256, (n_pages, 1, 16, 4), device=device, generator=g).to(torch.uint8) for _ in "kv"]
    state = [torch.from_numpy(x).to(device) for x in (table, np.array(lens, np.int32), refs)]
    ws = {}
    for parents in ([0] * rows, list(range(rows))[::-1], rng.integers(0, rows, rows).tolist()):
        run(device, tensors, state, parents, 16, ws)


def test_captured(device):
    announce("reorder, captured")
    tensors, state = make(device, 4, 6, 4, 16, [37, 20, 16, 40, 1, 33], 60)
    parents = torch.tensor([1, 1, 0, 5, 4, 4], device=device, dtype=torch.int32)
    keep = [t.clone() for t in (*tensors, *state)]
    ws = {}
    ia.reorder_sequences(tensors, *state, parents, page_size=16, workspace=ws)
    torch.cuda.synchronize()
    for t, k in zip((*tensors, *state), keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok = ia.reorder_sequences(tensors, *state, parents, page_size=16, workspace=ws)
    alone = torch.cuda.CUDAGraph()
    with torch.cuda.graph(alone):  # (with memory of its own)
        ok_too = ia.reorder_sequences(tensors, *state, parents, page_size=16)
    rng = np.random.default_rng(0)
    for step in range(4):
        parents.copy_(torch.from_numpy(rng.integers(0, 6, 6).astype(np.int32)))
        want = B.reorder(*(x.cpu().numpy() for x in state), parents.cpu().numpy(), 16)
        (alone if step % 2 else graph).replay()
        torch.cuda.synchronize()
        for got, w in zip((*state, ok_too if step % 2 else ok), want[:4]):
            assert np.array_equal(got.cpu().numpy(), w)


def test_refusals(device):
    tensors, (table, lens, refs) = make(device, 4, 4, 3, 16, [37, 20, 16, 40], 20)
    p = torch.zeros(4, device=device, dtype=torch.int32)
    for call in (lambda: ia.reorder_sequences(tensors, table, lens, refs, p[:3], page_size=16),
                 lambda: ia.reorder_sequences(tensors, table, lens, refs, p.long(), page_size=16),
                 lambda: ia.reorder_sequences(tensors, table, lens, refs, p, page_size=0),
                 lambda: ia.reorder_sequences(tensors, table, lens[:3], refs, p, page_size=16),
                 lambda: ia.reorder_sequences([t[:5] for t in tensors], table, lens, refs, p, page_size=16)):
        with pytest.raises(ValueError):
            call()
