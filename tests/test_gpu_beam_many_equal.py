"""Selections where many candidates have one key: rows that a mask leaves at the type's lowest value,
flat rows, beams that hold the same.  Places are checked exactly: equal keys go to the lower one.
(The bar of a score and of its order is that of the other tests of selection.)"""

import numpy as np
import pytest
import torch

import interattn_amd as ia
from oracle import beam as B
from tests._util import announce
from tests.test_gpu_beam_select import check

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
SIZES = [(1, 1, 700, 40), (1, 4, 32000, 8), (3, 8, 5003, 16), (2, 64, 3000, 64), (1, 33, 20000, 64), (40, 5, 9001, 10),
         (1, 2, 128000, 64)]


def places(got, beams, vocab):
    _, tok, par = (x.cpu().numpy().astype(np.int64) for x in got)
    return (par - np.arange(tok.shape[0])[:, None] * beams) * vocab + tok


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("allowed", [0, 1, 3])
@pytest.mark.parametrize("batch,beams,vocab,n", SIZES)
def test_rows_masked_to_the_lowest_value(device, dtype, allowed, batch, beams, vocab, n):
    """A grammar leaves a few tokens of a row (of some rows none): the others' keys are the lowest
    value, beside which a score counts for nothing, and fill the places that are left."""
    announce(f"beam select, masked {dtype} {allowed} {batch}x{beams} of {vocab}, {n}")
    g = torch.Generator(device=device)
    g.manual_seed(vocab + allowed)
    logits = torch.full((batch * beams, vocab), torch.finfo(dtype).min, device=device, dtype=dtype)
    for i in range(allowed):
        at = torch.randint(0, vocab, (batch * beams,), device=device, generator=g)
        rows = torch.arange(batch * beams, device=device)[i::2]
        logits[rows, at[i::2]] = (torch.randn(rows.shape, device=device, generator=g) * 3).to(dtype)
    scores = torch.randn((batch, beams), device=device, generator=g) * 4 - 20
    got = ia.beam_select(logits, scores, n)
    check(got, logits, scores, n)
    want = B.select(B.keys(logits.double().cpu().numpy(), scores.cpu().numpy()), n)
    assert np.array_equal(places(got, beams, vocab), want)


@pytest.mark.parametrize("batch,beams,vocab,n", SIZES)
def test_flat_rows_and_equal_beams(device, batch, beams, vocab, n):
    """Everything equal; one row for all beams; the two mixed, behind a few better ones."""
    announce(f"beam select, flat {batch}x{beams} of {vocab}, {n}")
    g = torch.Generator(device=device)
    g.manual_seed(vocab)
    scores = torch.full((batch, beams), -3.0, device=device)
    row = torch.randn((1, vocab), device=device, generator=g)
    some = torch.randint(0, 3, (1, vocab), device=device, generator=g).float()
    for x in (torch.zeros((batch * beams, vocab), device=device), row.repeat(batch * beams, 1),
              some.repeat(batch * beams, 1)):
        for dtype in (BF16, F32):
            logits = x.to(dtype)
            got = ia.beam_select(logits, scores, n)
            check(got, logits, scores, n)
            keys = B.keys(logits.double().cpu().numpy(), scores.cpu().numpy())
            assert np.array_equal(places(got, beams, vocab), B.select(keys, n))
    # keys below and above a crowd of equal ones, which is cut somewhere in its middle
    logits = some.repeat(batch * beams, 1)
    scores[:, beams // 2] += 2.0
    scores[:, :beams // 3] -= 1.0
    check(ia.beam_select(logits, scores, n), logits, scores, n)


def test_ended_beams_among_equal_ones(device):
    announce("beam select, ended beams among equal ones")
    scores = torch.full((2, 64), -2.0, device=device)
    done = torch.arange(128, device=device).view(2, 64) % 3 == 0
    logits = torch.zeros((128, 1), device=device)
    got = ia.beam_select(logits, scores, 60, done=done)
    check(got, logits, scores, 60, done)
    logits = torch.zeros((128, 900), device=device)
    scores[:, ::7] = -9.0
    for pad in (0, 899):
        got = ia.beam_select(logits, scores, 64, done=done, pad_token=pad)
        check(got, logits, scores, 64, done, pad)
