"""The 8-bit form of a matrix restated in numpy, in 64 bits: e4m3 values and e8m0 scales of blocks of 128.

Independent of the library: the e4m3 table is built from its definition (sign, 4 exponent bits with bias 7, 3 mantissa
bits, 0x7f and 0xff NaN, no infinities) and rounding is a search in that table, ties to the even code.
"""
from __future__ import annotations

import numpy as np


def _table() -> np.ndarray:
    t = np.zeros(128)
    for code in range(128):
        e, m = code >> 3, code & 7
        t[code] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
    t[127] = np.nan
    return t


POSITIVE = _table()
E4M3 = np.concatenate([POSITIVE, -POSITIVE])
E8M0 = np.array([2.0 ** (s - 127) for s in range(255)] + [np.nan])


def round_e4m3(v: np.ndarray) -> np.ndarray:
    """Codes of v (|v| <= 448) rounded to nearest, ties to even."""
    mag = np.abs(v)
    hi = np.clip(np.searchsorted(POSITIVE[:127], mag), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = mag - POSITIVE[lo], POSITIVE[hi] - mag
    code = np.where(below < above, lo, np.where(above < below, hi, np.where(lo % 2 == 0, lo, hi)))
    code = np.where(POSITIVE[hi] == mag, hi, code)
    return (code + np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def tops(v: np.ndarray, tile: bool) -> np.ndarray:
    """max|v| of every block."""
    rows, cols = v.shape
    r = 128 if tile else 1
    p = np.zeros((-(-rows // r) * r, -(-cols // 128) * 128))
    p[:rows, :cols] = np.abs(v)
    return p.reshape(p.shape[0] // r, r, p.shape[1] // 128, 128).max(axis=(1, 3))


def spread(s: np.ndarray, shape, tile: bool) -> np.ndarray:
    """A value per block as a value per element."""
    s = np.repeat(s, 128, axis=0)[: shape[0]] if tile else s
    return np.repeat(s, 128, axis=1)[:, : shape[1]]


def quantize(v: np.ndarray, tile: bool = False):
    """(codes, scale bytes) of finite or non-finite values in 64 bits."""
    v = np.asarray(v, dtype=np.float64)
    top = tops(v, tile)
    s = np.full(top.shape, 127)
    fine = np.isfinite(top)
    some = fine & (top > 0)
    s[some] = np.clip(127 + np.ceil(np.log2(top[some] / 448)).astype(int), 0, 254)
    s[some & (top > 448 * E8M0[s])] += 1  # log2's own rounding
    s[some & (s > 0) & (top <= 448 * E8M0[np.maximum(s - 1, 0)])] -= 1
    s[~fine] = 255
    per = spread(s, v.shape, tile)
    bad = per == 255
    codes = round_e4m3(np.where(bad, 0.0, np.where(bad, 0.0, v) / np.where(bad, 1.0, E8M0[per])))
    return np.where(bad, 127, codes).astype(np.uint8), s.astype(np.uint8)


def values(codes: np.ndarray, s: np.ndarray, tile: bool = False) -> np.ndarray:
    return E4M3[codes] * spread(E8M0[s], codes.shape, tile)
