"""Angles of far positions against frequencies times positions in whole numbers, with a pi that is
computed here: nothing of the expected angles comes from the plan."""

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import interattn_amd as ia
from tests._util import announce

FAR = [0, 1, -1, 2 ** 24, 10 ** 9 + 7, -123456789, 2 ** 31 - 1, -2 ** 31]


def _arctan_of_inverse(n, bits):
    """arctan(1 / n) in units of 2^-bits (a few hundred units off at most)."""
    total, power, k = 0, (1 << bits) // n, 0
    while power:
        total += (power if k % 2 == 0 else -power) // (2 * k + 1)
        power //= n * n
        k += 1
    return total


PI = Fraction(4 * (4 * _arctan_of_inverse(5, 300) - _arctan_of_inverse(239, 300)), 1 << 300)  # Machin


def turn_of(w, position):
    """The turn of ``position`` at ``w`` radians each, in [0, 1), as a fraction."""
    return Fraction(w) * position / (2 * PI) % 1


def apart(a, b):
    """Two turns' distance on the circle."""
    d = abs(a - b) % 1
    return min(d, 1 - d)


def frequencies():
    yarn = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)
    llama = dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192)
    yield dict(base=10000.0)
    yield dict(base=500000.0, scaling=llama)
    yield dict(base=10000.0, scaling=yarn)


@pytest.mark.parametrize("how", list(frequencies()), ids=["default", "llama3", "yarn"])
def test_turns_of_every_position(how):
    """A frequency is rounded once, to 2^-65 of a turn: its angle is 2^-34 off at the last position."""
    plan = ia.rotary_plan(128, device="cpu", **how)
    w, _ = ia.rotary_frequencies(128, **how)
    for x, t in zip(w, plan.turns.tolist()):
        for p in FAR:
            got = Fraction(p * t % (1 << 64), 1 << 64)
            assert apart(got, turn_of(x, p)) <= Fraction(abs(p), 1 << 65)


def test_any_frequency_that_is_given():
    """Negative ones, ones above a turn a position, large ones, ones below 2^-64 of a turn.  Whole
    turns a position are taken off in float64, whose 2 pi is off by 3.9e-17 of itself, below
    2^-54, for each of them."""
    w = [-0.75, 7.0, 6.283185307179586, 1e15, -3.7e30, 1e-300, 5e-19, 2.0 ** -60, 0.0, -1e-25]
    plan = ia.rotary_plan(2 * len(w), inv_freq=w, device="cpu")
    for x, t in zip(w, plan.turns.tolist()):
        whole = abs(Fraction(x)) // Fraction(2 * math.pi)  # (one of 6.283185307179586 itself)
        assert apart(Fraction(t % (1 << 64), 1 << 64), turn_of(x, 1)) <= Fraction(1, 1 << 65) + whole * Fraction(1, 1 << 54)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_rows(device, layout):
    """Rows at the ends of the range.  The kernel takes 2^-32 of a turn (cut off) of the angle:
    1.5e-9; its sums are off by 8 * 2^-24 of |a| + |b| at most, as at near positions."""
    announce(f"rotary, far rows {layout}")
    d = 128
    plan = ia.rotary_plan(d, base=500000.0, layout=layout, device=device)
    w, _ = ia.rotary_frequencies(d, base=500000.0)
    g = torch.Generator(device=device)
    g.manual_seed(1)
    x = torch.randn((len(FAR), 3, d), device=device, generator=g)
    got, _ = ia.apply_rotary(x, None, torch.tensor(FAR, device=device, dtype=torch.int32), plan)
    torch.cuda.synchronize()
    angle = np.array([[float(turn_of(f, p)) for f in w] for p in FAR])[:, None] * (2 * np.pi)
    v, y = x.double().cpu().numpy(), got.double().cpu().numpy()
    first, second = (slice(0, d // 2), slice(d // 2, d)) if layout == "half" else (slice(0, d, 2), slice(1, d, 2))
    a, b = v[..., first], v[..., second]
    bar = 8 * 2.0 ** -24 * (np.abs(a) + np.abs(b))
    assert (np.abs(y[..., first] - (a * np.cos(angle) - b * np.sin(angle))) <= bar).all()
    assert (np.abs(y[..., second] - (b * np.cos(angle) + a * np.sin(angle))) <= bar).all()
