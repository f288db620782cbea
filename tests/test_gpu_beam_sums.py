"""The logs of sums of beam selection, against 64 bits, where float32 loses most.

Of every term exp(x - M) the kernel forms, the argument's three roundings (the difference, its
product with log2 e, that constant itself) are off by 2.25 * 2^-24 of the argument, the exp
instruction by its last place, 2 * 2^-24.  A slice's reference lies at most 1 below its running
maximum, so a term's argument and the steps of the reference behind it are at most the term's
depth M - x and twice 1.  A step's exp is off by its last place too, but what is behind it has
lost a factor e by then: 1.2 of them count at most.  32 terms are joined in 5 additions (bf16; 16 in 4).
Together, with D the depth of a row's tokens averaged by their probability:

    2^-24 (2.25 (D + 2) + 2 + 2 * 1.2 + 5)  <=  2^-24 (14 + 2.3 D),

the rest is in 64 bits; a returned score is rounded once more, 2^-24 of itself."""

import pytest
import torch

import interattn_amd as ia
from tests._util import announce

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = 2.0 ** -24


def errors(logits, beams, n):
    """``(|score - its value in 64 bits|, the value)`` of the n best, and the deepest row's D."""
    scores = torch.zeros((logits.shape[0] // beams, beams), device=logits.device)
    got, tokens, parents = ia.beam_select(logits, scores, n)
    x = logits.double()
    logp = torch.log_softmax(x, -1)
    depth = (logp.exp() * (x.amax(-1, keepdim=True) - x)).sum(-1).max().item()
    want = logp[parents.long().flatten(), tokens.long().flatten()].view(got.shape)
    return (got.double() - want).abs(), want, depth


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("first,peak", [(3.5, 11.2), (0.3, 8.1), (-2.0, 5.7)])
def test_a_late_token_that_dominates(device, dtype, first, peak):
    """Slices that begin with one maximum and hold a far larger token later, the rest far below:
    the token is nearly the whole sum (D below 0.5), so its own term has to be right."""
    announce(f"beam sums, late peak {dtype} {first} {peak}")
    g = torch.Generator(device=device)
    g.manual_seed(round(100 * peak))
    rows, vocab = 512, 128000
    x = torch.full((rows, vocab), -40.0, device=device)
    x[:, ::1000] = first + 0.2 * torch.rand((rows, vocab // 1000), device=device, generator=g)
    at = torch.randint(0, vocab, (rows,), device=device, generator=g)
    x[torch.arange(rows, device=device), at] = peak + 0.2 * torch.rand((rows,), device=device, generator=g)
    off, want, depth = errors(x.to(dtype), 8, 8)
    assert depth < 0.5
    assert bool((off <= 2.0 ** -21 + HALF_STEP * want.abs()).all()), (off.max().item() * 2 ** 21)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("above", [0.0, 1.3, 4.7, 8.9, 9.7, 11.3, 14.1])
def test_a_flat_row_with_a_peak(device, dtype, above):
    """Equal terms, whose roundings are the same, with most of the sum ``above`` under the maximum."""
    announce(f"beam sums, flat rows {dtype} {above}")
    rows, vocab = 96, 128001
    level = torch.linspace(-7.3, 6.1, rows, device=device)
    x = level[:, None].repeat(1, vocab)
    x[torch.arange(rows, device=device), torch.arange(rows, device=device) * 1301 + 7] += above
    off, want, depth = errors(x.to(dtype), 4, 4)
    assert bool((off <= HALF_STEP * (14 + 2.3 * depth + want.abs())).all()), (off.max().item() / HALF_STEP, depth)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_rows_that_rise_slowly(device, dtype):
    """The reference moves with nearly every group; equal values in stretches."""
    announce(f"beam sums, rising rows {dtype}")
    vocab = 60000
    step = torch.arange(vocab, device=device) // 2048
    x = torch.stack([step * s for s in (0.3, 0.77, 0.999, 1.001, 1.7, 3.1, 7.9, 8.1)])
    for y in (x, x.flip(1)):
        off, want, depth = errors(y.to(dtype), 2, 5)
        assert bool((off <= HALF_STEP * (14 + 2.3 * depth + want.abs())).all()), (off.max().item() / HALF_STEP, depth)


def test_rows_that_differ_by_a_constant_tie(device):
    """Shifted rows have equal keys, so the lower place comes first, whatever the shift."""
    announce("beam sums, shifted rows")
    g = torch.Generator(device=device)
    g.manual_seed(4)
    row = torch.randint(-(1 << 12), 1 << 12, (30000,), device=device, generator=g).float() / 1024
    row[torch.randint(0, 30000, (40,), device=device, generator=g)] += 3.0
    # (whole numbers of 2^-10 below 2^13: the shifted rows are exact)
    x = torch.stack([row + s for s in (0.0, 1.0, 4096.0, -2048.0, 0.0078125, 100.0, 8000.0, -31.0)])
    for order in (list(range(8)), [2, 6, 0, 3, 1, 4, 5, 7]):
        s, tok, par = ia.beam_select(x[order], torch.zeros((1, 8), device=device), 8)
        assert par.tolist() == [list(range(8))] and len(set(tok[0].tolist())) == 1
        assert len(set(s[0].tolist())) == 1
