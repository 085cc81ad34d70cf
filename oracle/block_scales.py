"""A paged e4m3 cache with a scale for each block of tokens and head, in float64
(oracle; test only).  No counterpart in the reference.

* code c of cache row ``slot``, head h stands for ``c * scale[slot // unit, h]``;
* the scale that an append gives a block is ``power(amax)``: the smallest power of
  two, from 2^-60 to 2^60, with ``amax <= 448 * it``, amax the largest finite
  magnitude of the call's rows in the block -- or the old scale, if that is larger
  and the rows do not hold the block's first token;
* codes are the nearest e4m3 values (ties to even, saturating, NaN kept) of
  value / scale; where the scale grew, the codes before the call's rows are
  e4m3(code * old / new).

Pinned by ``tests/test_oracle_block_scales.py``.
"""
from __future__ import annotations

import math

import numpy as np

from .fp8 import decode_e4m3fn, encode_e4m3fn


def power(amax: float) -> float:
    if amax == 0:
        return 2.0 ** -60
    m, e = math.frexp(amax)    # amax = m * 2^e, 448 = 0.875 * 2^9
    return 2.0 ** min(60, max(-60, e - 9 + (m > 0.875)))


def encode(y):
    """Codes (uint8) of float64 values.  Rounded to odd in float32 first, so that the codes are those of the float64."""
    y = np.clip(np.asarray(y, dtype=np.float64), -448.0, 448.0)
    f = y.astype(np.float32)
    back = f.astype(np.float64)
    toward = np.where(back > y, np.float32(-np.inf), np.float32(np.inf))
    odd = np.where(back == y, f, np.where(f.view(np.uint32) & 1, f, np.nextafter(f, toward, dtype=np.float32)))
    return encode_e4m3fn(np.where(np.isnan(y), f, odd).astype(np.float32))


def transform(x, weight=None, offset=1.0, eps=1e-6, cos_sin=None, positions=None, rot=0):
    """Rows ``x [N, H, D]`` normed and rotated, float64; NaN rows for positions outside the table."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (np.asarray(weight, dtype=np.float64) + offset)
    if rot:
        table = np.asarray(cos_sin, dtype=np.float64).reshape(-1, rot)
        pos = np.asarray(positions)
        bad = (pos < 0) | (pos >= len(table))
        row = table[np.where(bad, 0, pos)][:, None]
        c, s = row[..., :rot // 2], row[..., rot // 2:]
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        x = np.concatenate([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
        x[bad] = np.nan
    return x


def append(z, codes, scales, slots, unit):
    """Appends ``z [N, H, D]`` (float64): new ``(codes [S, H, D] uint8, scales [S / unit, H])`` of the flat cache."""
    codes, scales = codes.copy(), scales.astype(np.float64)
    rows: dict[int, list[int]] = {}
    for i, s in enumerate(np.asarray(slots).tolist()):
        if 0 <= s < len(codes):
            rows.setdefault(s // unit, []).append(i)
    for block, idx in rows.items():
        first = min(int(slots[i]) for i in idx) - block * unit
        for h in range(z.shape[1]):
            x = np.abs(z[idx, h])
            need = power(float(np.max(x[np.isfinite(x)], initial=0.0)))
            old = float(scales[block, h])
            new = need if first == 0 else max(old, need)
            if first and new > old:
                at = slice(block * unit, block * unit + first)
                codes[at, h] = encode(decode_e4m3fn(codes[at, h]).astype(np.float64) * (old / new))
            for i in idx:
                codes[int(slots[i]), h] = encode(z[i, h] / new)
            scales[block, h] = new
    return codes, scales.astype(np.float32)


def values(codes, scales, unit):
    """Float64 values of a flat cache ``[S, H, D]``."""
    return decode_e4m3fn(codes).astype(np.float64) * np.repeat(scales.astype(np.float64), unit, 0)[:, :, None]
