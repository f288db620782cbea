"""Rotary positions in 64 bits: rows turned by their positions' angles."""

import numpy as np


def turn(x, positions, inv_freq, layout="half", factor=1.0, inverse=False):
    """``x [tokens, heads, D]`` with its first ``2 * len(inv_freq)`` channels turned."""
    x = np.asarray(x, np.float64)
    w = np.asarray(inv_freq, np.float64)
    r = 2 * len(w)
    angle = np.asarray(positions, np.float64)[:, None, None] * w
    c, s = np.cos(angle) * factor, np.sin(angle) * factor * (-1.0 if inverse else 1.0)
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])
    with np.errstate(invalid="ignore"):
        first, second = a * c - b * s, b * c + a * s
    out = x.copy()
    if layout == "half":
        out[..., :r // 2], out[..., r // 2:r] = first, second
    else:
        out[..., 0:r:2], out[..., 1:r:2] = first, second
    return out
