"""Beam search's selection against the order of keys in 64 bits.

Bar of a score: exp in float32 is off by 2^-22 relative at most (its argument's rounding,
2^-24 |x - M| log2 e for the terms that count, and the instruction's last place), so the log of a
sum by 2^-21; a returned score is rounded once more, 2^-24 of itself.  Tokens are equal unless two
keys are closer than that bar, which no listed case is by chance: equal keys are made so on
purpose, and go to the lower place.  That holds inside a row and between rows that hold the same
values in the same order (up to a constant); two rows of the same values in another order have
logs of sums that are each off by up to 2^-21, so which of them comes first is not theirs to say."""

import math

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import beam as B
from tests._util import announce

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def check(got, logits, scores, n, done=None, pad=0):
    torch.cuda.synchronize()
    s, tok, par = (x.cpu().numpy() for x in got)
    vocab = logits.shape[1]
    keys = B.keys(logits.double().cpu().numpy(), scores.cpu().numpy(), None if done is None else done.cpu().numpy(), pad)
    place = B.select(keys, n)
    want = np.take_along_axis(keys, place, 1)
    batch, beams = scores.shape
    at = (par - np.arange(batch)[:, None] * beams).astype(np.int64) * vocab + tok
    assert ((par // beams) == np.arange(batch)[:, None]).all() and (tok >= 0).all() and (tok < vocab).all()
    assert np.array_equal(np.isinf(s), np.isinf(want.astype(np.float32)))
    fine = np.isfinite(want)
    bar = 2.0 ** -21 + 2.0 ** -24 * np.abs(want[fine])
    assert (np.abs(s[fine] - want[fine]) <= bar).all()
    # a place differs only where the keys do not tell (never equal ones)
    mine = np.take_along_axis(keys, at, 1)
    differ = at != place
    x = logits.double().cpu().numpy().reshape(batch, beams, vocab)
    with np.errstate(invalid="ignore"):
        x = x - x.max(-1, keepdims=True)
    for b, i in np.argwhere(differ & (mine == want)):
        j, k = at[b, i] // vocab, place[b, i] // vocab
        assert not np.array_equal(x[b, j], x[b, k], equal_nan=True), "equal keys go to the lower place"
    assert (np.abs(mine[differ] - want[differ]) <= 2.0 ** -20).all()
    assert all(len(set(r)) == n for r in at)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("batch,beams,vocab,n,pad_cols", [
    (1, 1, 1, 1, 0), (1, 1, 7, 7, 0), (3, 2, 5, 10, 1), (1, 4, 32000, 8, 0), (2, 5, 50021, 5, 3), (2, 1, 513, 64, 7),
    (1, 64, 1000, 64, 0), (5, 3, 511, 3, 0), (40, 8, 2049, 16, 1), (1, 2, 131072, 33, 0),
    (2100, 1, 4100, 5, 0), (800, 3, 5001, 7, 2), (300, 1, 20000, 16, 0), (24, 7, 30000, 64, 0),
])
def test_best_continuations(device, dtype, batch, beams, vocab, n, pad_cols):
    """Odd vocabularies, rows that begin at any element."""
    announce(f"beam select {dtype} {batch}x{beams} of {vocab}, {n} best")
    g = torch.Generator(device=device)
    g.manual_seed(vocab + n)
    rows = batch * beams
    # float32 values that bf16 holds apart are continuous: ties only where bf16 makes them
    buf = (torch.randn((rows * (vocab + pad_cols) + 1,), device=device, generator=g) * 3).to(dtype)[1:]
    logits = buf.view(rows, vocab + pad_cols)[:, :vocab]
    scores = torch.randn((batch, beams), device=device, generator=g) * 4 - 20
    check(ia.beam_select(logits, scores, n), logits, scores, n)
    ws = {}
    for _ in range(2):
        again = ia.beam_select(logits, scores, n, workspace=ws)
    check(again, logits, scores, n)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_equal_keys_go_to_the_lower_place(device, dtype):
    """All logits equal, beams with equal rows, one value at many places, both zeros."""
    announce(f"beam select, ties {dtype}")
    for vocab, n in ((40, 9), (3001, 64), (20000, 24)):
        logits = torch.zeros((6, vocab), device=device, dtype=dtype)
        scores = torch.full((2, 3), -1.0, device=device)
        s, tok, par = ia.beam_select(logits, scores, n)
        torch.cuda.synchronize()
        assert tok.tolist() == [list(range(n))] * 2 and par.tolist() == [[0] * n, [3] * n]
        logits[:, vocab // 2] = 5.0
        logits[:, vocab // 2 + 7] = 5.0
        logits[:, ::3] = -0.0
        check(ia.beam_select(logits, scores, n), logits, scores, n)
        check(ia.beam_select(logits, scores, 6), logits, scores, 6)
        g = torch.Generator(device=device)
        g.manual_seed(vocab)
        few = torch.randint(0, 4, (6, vocab), device=device, generator=g).to(dtype)
        check(ia.beam_select(few, scores, n), few, scores, n)
        rising = (torch.arange(6 * vocab, device=device).view(6, vocab) // 50).to(F32).div(16).to(dtype)
        check(ia.beam_select(rising, scores, n), rising, scores, n)


def test_more_equal_keys_than_fit(device):
    """64 beams of equal rows, the best 64: thousands of keys reach the threshold."""
    announce("beam select, 64 equal beams")
    g = torch.Generator(device=device)
    g.manual_seed(6)
    scores = torch.full((2, 64), -3.0, device=device)
    row = torch.randn((1, 3000), device=device, generator=g)
    for logits in (row.expand(128, 3000), torch.zeros((128, 3000), device=device), row.bfloat16().repeat(128, 1)):
        check(ia.beam_select(logits, scores, 64), logits, scores, 64)


@pytest.mark.parametrize("n", [1, 3, 16])
def test_best_that_lie_in_one_slice(device, n):
    """All of a row's best at its end, at its start, and one equal value in every stretch: what the
    slices of a row learn of each other must not cost a candidate."""
    announce(f"beam select, uneven slices, {n} best")
    g = torch.Generator(device=device)
    g.manual_seed(n)
    logits = torch.randn((4 * 3, 60000), device=device, generator=g)
    logits[0, -40:] += 30
    logits[1, :40] += 30
    logits[2, 5::997] = 9.0
    logits[3] = logits[3].sort().values
    logits[4] = logits[4].sort(descending=True).values
    logits[5, 30000:30040] = 20.0
    logits[6:9] = logits[2] + torch.tensor([[0.0], [1.0], [-2.0]], device=device)
    logits[9, ::2] = -1e30
    scores = torch.zeros((4, 3), device=device)
    for x in (logits, logits.bfloat16()):
        check(ia.beam_select(x, scores, n), x, scores, n)


def test_what_offers_nothing(device):
    """-inf and NaN logits, beams of -inf or NaN scores, rows that reach +inf, rows of -inf."""
    announce("beam select, nothing offered")
    g = torch.Generator(device=device)
    g.manual_seed(3)
    for dtype in (BF16, F32):
        logits = torch.randn((12, 700), device=device, generator=g).to(dtype)
        scores = torch.randn((3, 4), device=device, generator=g)
        logits[0, 5:600] = -math.inf
        logits[1] = -math.inf
        logits[2, 3] = math.inf
        logits[3, 100:300] = math.nan
        logits[4:8] = -math.inf
        logits[8, 1:] = -math.inf
        logits[9:12] = math.nan
        scores[2, 3] = math.nan
        for n in (4, 8, 30):
            check(ia.beam_select(logits, scores, n), logits, scores, n)
        first = torch.full((3, 4), -math.inf, device=device)
        first[:, 0] = 0
        check(ia.beam_select(logits, first, 8), logits, first, 8)
        lows = logits.clone()
        lows[:] = torch.finfo(dtype).min
        check(ia.beam_select(lows, scores, 6), lows, scores, 6)


@pytest.mark.parametrize("n", [1, 4, 12])
def test_beams_that_have_ended(device, n):
    announce(f"beam select, ended beams {n}")
    g = torch.Generator(device=device)
    g.manual_seed(n)
    logits = torch.randn((5 * 4, 999), device=device, generator=g).bfloat16()
    scores = torch.randn((5, 4), device=device, generator=g) * 3 - 6
    done = torch.zeros((5, 4), dtype=torch.bool, device=device)
    done[0, 1] = done[1, :] = True
    done[2, 2:] = True
    scores[2, 2] = 50.0
    scores[1, 3] = -math.inf
    logits[4:8] = math.nan  # (not read)
    for pad in (0, 998, 17):
        got = ia.beam_select(logits, scores, n, done=done, pad_token=pad)
        check(got, logits, scores, n, done, pad)


def test_wide_spreads_keep_their_sums(device):
    """A maximum that comes late, rows that rise by 100 units, one dominating token."""
    announce("beam select, sums")
    x = torch.linspace(-60, 60, 30011, device=device).repeat(4, 1)
    x[1] = x[1].flip(0)
    x[2, 12345] = 300.0
    x[3] = -1e4
    scores = torch.zeros((2, 2), device=device)
    for logits in (x, x.bfloat16()):
        check(ia.beam_select(logits, scores, 5), logits, scores, 5)


def test_a_captured_selection(device):
    announce("beam select, captured")
    g = torch.Generator(device=device)
    g.manual_seed(5)
    logits, scores = torch.randn((8, 4000), device=device, generator=g), torch.zeros((2, 4), device=device)
    ws = {}
    ia.beam_select(logits, scores, 8, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ia.beam_select(logits, scores, 8, workspace=ws)
    alone = torch.cuda.CUDAGraph()
    with torch.cuda.graph(alone):  # (with memory of its own)
        out += ia.beam_select(logits, scores, 8)
    for _ in range(3):
        logits.normal_(generator=g)
        scores.normal_(generator=g)
        want = ia.beam_select(logits, scores, 8)
        graph.replay()
        alone.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want * 2))


def test_refusals(device):
    x, s = torch.zeros((8, 100), device=device), torch.zeros((2, 4), device=device)
    done = torch.zeros((2, 4), dtype=torch.bool, device=device)
    for call in (lambda: ia.beam_select(x, s, 0), lambda: ia.beam_select(x, s, 65), lambda: ia.beam_select(x[:7], s),
                 lambda: ia.beam_select(x.half(), s), lambda: ia.beam_select(x, s.double()),
                 lambda: ia.beam_select(x.t().contiguous().t(), s), lambda: ia.beam_select(x, s, pad_token=100),
                 lambda: ia.beam_select(x, s, pad_token=-1), lambda: ia.beam_select(x, s, done=done.int()),
                 lambda: ia.beam_select(x, s, done=done[:1]), lambda: ia.beam_select(x[:, :3], s, 13),
                 lambda: ia.beam_select(x, s.t().contiguous().t())):
        with pytest.raises(ValueError):
            call()
    out = ia.beam_select(x[:0], s[:0], 3)
    assert [tuple(o.shape) for o in out] == [(0, 3)] * 3
