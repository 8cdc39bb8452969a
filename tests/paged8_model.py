"""Plain implementations of what is stored in 8-bit pages, number by number."""
from __future__ import annotations

import numpy as np

BLOCK = 16
NAN = 0x7F


def e4m3_table():
    """The magnitudes of e4m3's codes 0 .. 126, in float64."""
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9.0)


TABLE = e4m3_table()


def nearest(x):
    """Codes of the nearest e4m3 numbers, ties to the even code, of |x| <= 448;
    NAN for what is not finite."""
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(TABLE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    down, up = a - TABLE[lo], TABLE[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = code | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isfinite(x), code, NAN)


def value(code):
    mag = np.append(TABLE, np.nan)[code & 0x7F]
    return np.where(code & 0x80, -mag, mag)


def unit(top):
    """Exponent of the smallest power of two from 2^-15 on that `top` is at
    most 448 of."""
    k = -15
    while top > 448.0 * 2.0 ** k:
        k += 1
    return k


def store(codes, k, held, new):
    """`new` rows [n][128] (float64, f16 numbers) behind the first `held` of a
    block [16][128] whose unit is 2^k: its codes and exponent afterwards."""
    codes = codes.copy()
    fine = np.abs(new[np.isfinite(new)])
    need = unit(fine.max() if fine.size else 0.0)
    now = max(k, need) if held else need
    if held and now > k:
        codes[:held] = canon(nearest(value(codes[:held]) * 2.0 ** (k - now)))
    most = 240.0 if now == 8 else 448.0
    scaled = new * 2.0 ** -now
    codes[held:held + len(new)] = nearest(np.where(np.isfinite(scaled), np.clip(scaled, -most, most), np.nan))
    return codes, now


def canon(codes):
    """NaN has two codes: one of them."""
    return np.where((codes & 0x7F) == NAN, NAN, codes)
