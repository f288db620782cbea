"""Page copying, forking, reserving, freeing and compacting against the same rules in plain
Python: tables, lengths, counts and page contents are equal, whole."""

import random

import pytest
import torch

import interattn_amd as ia
from tests._util import announce

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ the rules

class Model:
    """Host copy of a cache's state, with the rules of the calls."""

    def __init__(self, table, lens, refs, pools, page):
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)
        self.pools, self.page = [p.clone() for p in pools], page

    def lowest(self, n):
        return [i for i, r in enumerate(self.refs) if r == 0][:n]

    def free(self, rows):
        for row in dict.fromkeys(r for r in rows if 0 <= r < len(self.lens)):
            for c, pg in enumerate(self.table[row]):
                if 0 <= pg < len(self.refs):
                    self.refs[pg] -= 1
                self.table[row][c] = -1
            self.lens[row] = 0

    def fork(self, src, dst):
        ok, copies = [], []
        exists = lambda r: 0 <= r < len(self.lens)  # noqa: E731
        avail = self.lowest(len(src))
        start = [list(r) for r in self.table]
        for i, (s, d) in enumerate(zip(src, dst)):
            good = exists(s) and exists(d) and s not in dst and d not in dst[:i]
            good = good and self.lens[d] == 0 and all(pg < 0 for pg in start[d])
            part = good and self.lens[s] % self.page
            good = good and self.lens[s] <= len(start[s]) * self.page
            if good and part:
                old = start[s][self.lens[s] // self.page]
                good = 0 <= old < len(self.refs) and bool(avail)
            ok.append(int(bool(good)))
            if not good:
                continue
            whole = self.lens[s] // self.page
            for c in range(whole):
                self.table[d][c] = start[s][c]
                if 0 <= start[s][c] < len(self.refs):
                    self.refs[start[s][c]] += 1
            if part:
                new = avail.pop(0)
                self.table[d][whole] = new
                self.refs[new] = 1
                copies.append((old, new))
            self.lens[d] = self.lens[s]
        for a, b in copies:
            for p in self.pools:
                p[b] = p[a]
        return ok

    def reserve(self, grow):
        ok, avail = [], self.lowest(len(self.refs))
        for row, g in enumerate(grow):
            n = self.lens[row]
            if g <= 0:
                ok.append(1)
                continue
            if n < 0 or n + g > len(self.table[row]) * self.page:
                ok.append(0)
                continue
            at = [c for c in range(n // self.page, -(-(n + g) // self.page)) if self.table[row][c] < 0]
            if len(at) > len(avail):
                ok.append(0)
                continue
            for c in at:
                self.table[row][c] = avail.pop(0)
                self.refs[self.table[row][c]] = 1
            ok.append(1)
        return ok

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        movers = [i for i, r in enumerate(self.refs) if r > 0 and i >= live]
        holes = [i for i, r in enumerate(self.refs) if r <= 0 and i < live]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for p in self.pools:
                p[b] = p[a]
        self.table = [[to.get(pg, pg) for pg in row] for row in self.table]
        return live


def state(device, seed, rows, cols, page, n_pages, pools, used=0.6):
    """A random consistent cache: some rows share whole pages, some are empty, some hold
    pages past their length."""
    r = random.Random(seed)
    ids = list(range(n_pages))
    r.shuffle(ids)
    budget = int(n_pages * used)
    table, lens, refs = [], [], [0] * n_pages
    for row in range(rows):
        entry, n = [-1] * cols, 0
        if row and r.random() < 0.3 and lens[row - 1] >= page:
            n = lens[row - 1] // page * page
            entry[:n // page] = table[row - 1][:n // page]
        elif r.random() < 0.8 and budget:
            held = r.randint(1, min(cols, budget))
            budget -= held
            entry[:held] = [ids.pop() for _ in range(held)]
            n = r.randint(max(0, (held - 2) * page), held * page)
        for pg in entry:
            if pg >= 0:
                refs[pg] += 1
        table.append(entry)
        lens.append(n)
    dev = dict(table=torch.tensor(table, device=device, dtype=torch.int32),
               lens=torch.tensor(lens, device=device, dtype=torch.int32),
               refs=torch.tensor(refs, device=device, dtype=torch.int32))
    return dev, Model(table, lens, refs, pools, page)


def make_pools(device, n_pages, hkv, page, d, kinds, seed):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    out = []
    for kind in kinds:
        if kind == "paired":
            buf = torch.randn((n_pages, hkv, 2, page, d), device=device, generator=gen).to(torch.bfloat16)
            out += [buf[:, :, 0], buf[:, :, 1]]
        elif kind == "fp8":
            out.append(torch.randn((n_pages, hkv, page, d), device=device, generator=gen).to(torch.float8_e4m3fn)
                       .view(torch.uint8))
            out.append(torch.rand((n_pages, hkv), device=device, generator=gen))
        elif kind == "tokens":  # a pool whose tokens lie outside its heads
            out.append(torch.randn((n_pages, page, hkv, d), device=device, generator=gen).permute(0, 2, 1, 3))
        else:
            out.append(torch.randn((n_pages, hkv, page, d), device=device, generator=gen).to(torch.bfloat16))
    return out


def same(dev, pools, model, what):
    torch.cuda.synchronize()
    assert dev["refs"].tolist() == model.refs, (what, "refs")
    assert dev["lens"].tolist() == model.lens, (what, "lens")
    assert dev["table"].tolist() == model.table, (what, "table")
    for i, (a, b) in enumerate(zip(pools, model.pools)):
        assert torch.equal(a, b), (what, "pool", i)


KINDS = [["bf16"], ["paired"], ["fp8", "fp8"], ["tokens", "bf16", "paired"], []]


@pytest.mark.parametrize("seed", range(10))
def test_random_life(seed, device):
    """A random run of every call on one state, checked after each."""
    announce(f"pages life {seed}")
    r = random.Random(seed)
    page, rows, cols = r.choice([1, 16, 16, 48]), r.choice([3, 9, 20]), r.choice([1, 5, 70, 300])
    n_pages = r.choice([4, 61, 256, 1029, 5000])
    pools = make_pools(device, n_pages, 2, 4, 16, KINDS[seed % len(KINDS)], seed)
    dev, model = state(device, seed, rows, cols, page, n_pages, pools)
    ws = {}
    i32 = lambda x: torch.tensor(x, device=device, dtype=torch.int32)  # noqa: E731
    for step in range(12):
        call = r.choice(["free", "fork", "fork", "reserve", "reserve", "compact", "grow"])
        if call == "free":
            some = [r.randrange(-1, rows + 1) for _ in range(r.randint(1, 4))]
            model.free(some)
            ia.free_sequences(dev["table"], dev["lens"], dev["refs"], i32(some))
        elif call == "fork":
            n = r.randint(1, 6)
            src, dst = [r.randrange(-1, rows + 1) for _ in range(n)], [r.randrange(-1, rows + 1) for _ in range(n)]
            want = model.fork(src, dst)
            ok = ia.fork_sequences(pools, dev["table"], dev["lens"], dev["refs"], i32(src), i32(dst), page_size=page,
                                   workspace=ws)
            assert ok.tolist() == want, (seed, step, src, dst)
        elif call == "reserve":
            grow = [r.choice([0, 0, 1, page, 3 * page + 1, -5, cols * page]) for _ in range(rows)]
            want = model.reserve(grow)
            ok = ia.reserve_pages(dev["table"], dev["lens"], dev["refs"], i32(grow), page_size=page, workspace=ws)
            assert ok.tolist() == want, (seed, step, grow)
        elif call == "compact":
            want = model.compact()
            assert ia.compact_pages(pools, dev["table"], dev["refs"], workspace=ws).tolist() == [want]
        else:  # rows grow into the pages they have
            for row in range(rows):
                held = sum(pg >= 0 for pg in model.table[row])
                if r.random() < 0.5 and model.lens[row] < held * page:
                    model.lens[row] += r.randint(0, held * page - model.lens[row])
            dev["lens"].copy_(i32(model.lens))
        same(dev, pools, model, (seed, step, call))


def test_short_of_pages_serves_what_it_can(device):
    announce("pages short")
    page, n_pages = 16, 6
    pools = make_pools(device, n_pages, 1, page, 16, ["bf16"], 0)
    i32 = lambda x: torch.tensor(x, device=device, dtype=torch.int32)  # noqa: E731
    table = [[0, 1, -1, -1], [-1] * 4, [-1] * 4, [-1] * 4, [-1] * 4]
    dev = dict(table=i32(table), lens=i32([20, 0, 0, 0, 0]), refs=i32([1, 1, 0, 0, 0, 0]))
    model = Model(table, [20, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], pools, page)
    # three pages for row 1, three more for row 2 (one is left), one for row 3, none for row 4
    grow = [0, 40, 33, 16, 1]
    assert model.reserve(grow) == [1, 1, 0, 1, 0]
    assert ia.reserve_pages(dev["table"], dev["lens"], dev["refs"], i32(grow), page_size=page).tolist() == [1, 1, 0, 1, 0]
    same(dev, pools, model, "reserve")
    # a fork needs a page for the prompt's partial one: none is left until a row is freed
    assert ia.fork_sequences(pools, dev["table"], dev["lens"], dev["refs"], i32([0]), i32([2]), page_size=page).tolist() == [0]
    assert model.fork([0], [2]) == [0]
    same(dev, pools, model, "fork refused")
    ia.free_sequences(dev["table"], dev["lens"], dev["refs"], i32([3, 3]))
    model.free([3, 3])
    assert ia.fork_sequences(pools, dev["table"], dev["lens"], dev["refs"], i32([0, 0]), i32([2, 4]),
                             page_size=page).tolist() == model.fork([0, 0], [2, 4]) == [1, 0]
    same(dev, pools, model, "fork")


@pytest.mark.parametrize("kinds", [["bf16"] * 3, ["fp8"] * 2, ["paired"] * 30], ids=["bf16", "fp8", "60 tensors"])
def test_copy(kinds, device):
    announce(f"copy pages {kinds[0]} {len(kinds)}")
    n_pages = 40
    pools = make_pools(device, n_pages, 3, 16, 64, kinds, 1)
    want = [p.clone() for p in pools]
    src, dst = [3, 3, 39, -1, 5, 12, 40], [0, 1, 2, 4, 99, 12, 6]
    for s, d in ((3, 0), (3, 1), (39, 2)):
        for p in want:
            p[d] = p[s]
    ia.copy_pages(pools, torch.tensor(src, device=device, dtype=torch.int32),
                  torch.tensor(dst, device=device, dtype=torch.int32))
    torch.cuda.synchronize()
    for a, b in zip(pools, want):
        assert torch.equal(a, b)


def test_calls_replay_in_a_graph(device):
    """free, fork and reserve captured once, replayed on changing states, with eager calls of
    other sizes between."""
    announce("pages graph")
    page, n_pages, rows = 16, 300, 9
    pools = make_pools(device, n_pages, 2, page, 16, ["bf16"], 4)
    dev, model = state(device, 4, rows, 20, page, n_pages, pools)
    i32 = lambda x: torch.tensor(x, device=device, dtype=torch.int32)  # noqa: E731
    drop, src, dst, grow, ws = i32([5, 6]), i32([0, 1]), i32([5, 6]), i32([0] * 5 + [40, 3] + [0] * 2), {}

    def step():
        ia.free_sequences(dev["table"], dev["lens"], dev["refs"], drop)
        a = ia.fork_sequences(pools, dev["table"], dev["lens"], dev["refs"], src, dst, page_size=page, workspace=ws)
        return a, ia.reserve_pages(dev["table"], dev["lens"], dev["refs"], grow, page_size=page, workspace=ws)

    def expect(src_l, dst_l):
        model.free(drop.tolist())
        return model.fork(src_l, dst_l), model.reserve(grow.tolist())

    a, b = step()
    assert (a.tolist(), b.tolist()) == expect([0, 1], [5, 6])
    same(dev, pools, model, "eager")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph):
            a, b = step()
    torch.cuda.current_stream().wait_stream(side)
    for i, (x, y) in enumerate([(0, 1), (3, 3), (8, 2), (0, 5)]):
        src.copy_(i32([x, y]))
        graph.replay()
        torch.cuda.synchronize()
        assert (a.tolist(), b.tolist()) == expect([x, y], [5, 6]), i
        same(dev, pools, model, ("replay", i))
        ia.free_sequences(dev["table"], dev["lens"], dev["refs"], i32([7]))
        model.free([7])
        assert ia.fork_sequences(pools, dev["table"], dev["lens"], dev["refs"], i32([x]), i32([7]), page_size=page,
                                 workspace=ws).tolist() == model.fork([x], [7])
        assert ia.compact_pages(pools, dev["table"], dev["refs"], workspace=ws).tolist() == [model.compact()]
        same(dev, pools, model, ("between", i))
