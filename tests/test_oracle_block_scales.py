"""Pins oracle/block_scales.py: scales by their definition, codes by search, appends token by token."""
import numpy as np
import pytest

from oracle import block_scales as o
from oracle.fp8 import decode_e4m3fn

GRID = decode_e4m3fn(np.arange(127, dtype=np.uint8)).astype(np.float64)


@pytest.mark.parametrize("amax", [448.0, np.nextafter(448.0, 1e9), 447.9, 1.0, 1.75, 1.7500001, 3e-5, 2.0 ** -40, 6e8])
def test_power_is_the_smallest(amax):
    s = o.power(amax)
    assert np.log2(s) == int(np.log2(s))
    assert amax <= 448 * s and amax > 448 * s / 2


def test_power_stays_in_its_range():
    assert o.power(0.0) == o.power(1e-30) == 2.0 ** -60
    assert o.power(1e38) == 2.0 ** 60


def test_encode_is_the_nearest_code():
    r = np.random.default_rng(0)
    mid = (GRID[1:] + GRID[:-1]) / 2
    y = np.concatenate([r.normal(size=300) * 100, mid, np.nextafter(mid, 0), np.nextafter(mid, 1e9), [0.0, 500.0, -1e30]])
    got = o.encode(y)
    for v, c in zip(np.clip(y, -448, 448), got):
        d = np.abs(GRID - abs(v))
        best = np.flatnonzero(d == d.min())
        want = best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]
        assert (c & 0x7F) == want and (c >> 7) == np.signbit(v), (v, c, want)
    assert (o.encode(np.array([np.nan])) & 0x7F) == 0x7F


@pytest.mark.parametrize("unit", [32, 64])
def test_append_in_one_call_or_token_by_token(unit):
    """The scales agree, and the values where no code fell below e4m3's normal range on the way."""
    r = np.random.default_rng(unit)
    n, h, d = 2 * unit - 5, 2, 16
    z = r.normal(size=(n, h, d)) * 2.0 ** r.integers(-3, 4, size=(n, 1, 1))
    z = np.where(np.abs(z) < 2.0 ** -4, 1.0, z)
    slots = np.arange(unit, unit + n)
    codes = r.integers(0, 126, size=(4 * unit, h, d)).astype(np.uint8)
    scales = np.full((4, h), 2.0 ** 30, np.float32)
    c1, s1 = o.append(z, codes, scales, slots, unit)
    c2, s2 = codes, scales
    for i in range(n):
        c2, s2 = o.append(z[i:i + 1], c2, s2, slots[i:i + 1], unit)
    assert np.array_equal(s1, s2)
    assert np.array_equal(c1, c2)
    v = o.values(c1, s1, unit)[slots]
    assert (np.abs(v - z) <= 2.0 ** -4 * np.abs(z)).all()
    rest = np.setdiff1d(np.arange(4 * unit), slots)
    assert np.array_equal(c1[rest], codes[rest]) and (s1[[0, 3]] == 2.0 ** 30).all()


def test_a_grown_scale_moves_exponents():
    codes = np.arange(256, dtype=np.uint8).reshape(32, 1, 8)[:31]
    codes = np.concatenate([codes, np.zeros((1, 1, 8), np.uint8)])
    c, s = o.append(np.full((1, 1, 8), 448.0 * 8), codes, np.ones((1, 1), np.float32), np.array([31]), 32)
    assert s[0, 0] == 8
    was, now = decode_e4m3fn(codes[:31]).astype(np.float64), o.values(c, s, 32)[:31]
    nan = np.isnan(was)
    assert np.array_equal(nan, np.isnan(now))
    exact = ~nan & (np.abs(was) >= 2.0 ** -6 * 8)
    assert (now[exact] == was[exact]).all()
    assert (np.abs(now - was)[~nan] <= 2.0 ** -10 * 8).all()


def test_what_is_not_finite_has_no_say_in_the_scale():
    z = np.array([1.0, np.inf, -np.inf, np.nan, 100.0, -5.0, 0.0, 2.0]).reshape(1, 1, 8)
    c, s = o.append(z, np.zeros((32, 1, 8), np.uint8), np.ones((1, 1), np.float32), np.array([0]), 32)
    assert s[0, 0] == o.power(100.0)
    v = o.values(c, s, 32)[0, 0]
    assert v[1] == 448 * s[0, 0] and v[2] == -448 * s[0, 0] and np.isnan(v[3]) and v[0] == 1.0


def test_rows_outside_the_pool_are_skipped():
    codes = np.zeros((32, 1, 8), np.uint8)
    c, s = o.append(np.ones((3, 1, 8)), codes, np.ones((1, 1), np.float32), np.array([-1, 32, 1000]), 32)
    assert (c == 0).all() and (s == 1).all()


def test_transform_against_a_loop():
    r = np.random.default_rng(3)
    x, w = r.normal(size=(3, 2, 32)), r.normal(size=32)
    table = r.normal(size=(7, 16))
    z = o.transform(x, w, 1.0, 1e-6, table, np.array([6, 0, 7]), 16)
    for n, p in ((0, 6), (1, 0)):
        for h in range(2):
            y = x[n, h] / np.sqrt(np.mean(x[n, h] ** 2) + 1e-6) * (w + 1)
            for e in range(8):
                c, s = table[p, e], table[p, 8 + e]
                assert np.isclose(z[n, h, e], y[e] * c - y[e + 8] * s, rtol=1e-12)
                assert np.isclose(z[n, h, e + 8], y[e + 8] * c + y[e] * s, rtol=1e-12)
            assert np.allclose(z[n, h, 16:], y[16:], rtol=1e-12)
    assert np.isnan(z[2]).all()
