"""An 8-bit cache as it is written: e4m3 codes and the pages' power-of-two scales."""

import numpy as np

LARGEST = 448.0
LEAST_SCALE = 2.0 ** -126


def _values():
    code = np.arange(256)
    e, m = (code >> 3) & 15, code & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where(code & 128, -v, v)
    v[[0x7F, 0xFF]] = np.nan
    return v


VALUES = _values()  # of each code


def encode(y):
    """The nearest e4m3 code of each value, ties to the even one; what is not finite, or would
    round past 448, is 0x7F."""
    y = np.asarray(y, np.float64)
    mag = VALUES[:0x7F]
    a = np.abs(np.where(np.isfinite(y), y, 0.0))
    hi = np.clip(np.searchsorted(mag, a), 1, 0x7E)
    lo = hi - 1
    up, down = mag[hi] - a, a - mag[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.signbit(y), code | 0x80, code)
    return np.where(np.isfinite(y) & (a <= 464), code, 0x7F).astype(np.uint8)


def page_scale(largest):
    s = LEAST_SCALE
    while largest > LARGEST * s:
        s *= 2
    return s


def write_page(codes, scale, lo, rows):
    """One head's page ``codes [page, D]`` with ``scale``, of which the first ``lo`` rows are
    earlier tokens, after ``rows [n, D]`` behind them.  Returns ``(codes, scale)``."""
    codes = codes.copy()
    rows = np.asarray(rows, np.float64)
    fine = np.abs(rows[np.isfinite(rows)])
    largest = float(fine.max()) if fine.size else 0.0
    s = page_scale(largest)
    if lo:
        if np.isfinite(scale) and scale >= LEAST_SCALE and largest <= np.float64(np.float32(LARGEST * np.float32(scale))):
            s = float(scale)
        else:
            # (the kernel's product is a float32)
            with np.errstate(over="ignore", invalid="ignore"):
                again = VALUES[codes[:lo]].astype(np.float32) * (np.float32(scale) / np.float32(s))
            codes[:lo] = encode(again)
    with np.errstate(over="ignore"):
        codes[lo:lo + len(rows)] = encode((rows.astype(np.float32) / np.float32(s)).astype(np.float64))
    return codes, np.float32(s)
