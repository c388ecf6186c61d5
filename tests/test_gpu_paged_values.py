"""The paged attention calls beside infinities, NaN and values far apart: every
output against the definition in 64 bits, infinities and NaN where it has them
and only there, the rest within the bounds of paged_ref.py."""
import numpy as np
import pytest

import paged_ref as R
from paged_ref import BF16, F16, F32
from test_gpu_paged import TYPES, Case, say, seed

pytestmark = pytest.mark.gpu


def compare(got, want, tol):
    """NaN and infinities at the same places, finite values within tol."""
    odd = ~np.isfinite(want)
    np.testing.assert_array_equal(got[odd], want[odd])
    err = np.abs(got[~odd] - want[~odd])
    assert np.isfinite(got[~odd]).all(), np.argwhere(~np.isfinite(got) & ~odd)[:4]
    assert (err <= tol[~odd]).all(), (np.argwhere(~odd)[~(err <= tol[~odd])][:4], err.max())


def rows_of(c, s):
    n, r0 = c.new[s], int(c.start[s])
    q = R.from_bits(R.to_bits(c.q, c.act), c.act)[r0:r0 + n, :c.H * c.D].reshape(n, c.H, c.D)
    return q, int(c.kv[s]) - n + np.arange(n)


def got_of(c, s):
    return c.got()[int(c.start[s]):int(c.start[s + 1]), :c.H * c.D].reshape(c.new[s], c.H, c.D)


# heads, KV heads, dims, cached, new: 16-row tiles, 64-row tiles, 128-row tiles, cut 128-row tiles
PREFILL = [(4, 2, 64, [0, 30], [170, 160]), (4, 2, 128, [0, 30], [170, 160]), (20, 20, 128, [40] * 30, [9] * 30),
           (32, 2, 128, [0, 30], [170, 160]), (64, 4, 64, [0, 30], [170, 160]),
           (20, 20, 128, [0, 0, 70, 0, 3], [200, 260, 130, 60, 200]),
           (40, 20, 64, [0, 0, 70], [200, 260, 130]), (32, 2, 128, [2200, 2000], [150, 140]),
           (40, 2, 64, [2200, 2000], [150, 140])]


def put_values(c, s, odd):
    """odd: (key, KV head, dim, value) of sequence s's V, the last where several name
    one element; its keys, and V with zeros there."""
    k, v = c.pool.get(s, int(c.kv[s]))
    v, zeroed = v.copy(), v.copy()
    for j, g, d, x in odd:
        v[j, g, d], zeroed[j, g, d] = x, 0
    c.pool.put(s, np.arange(len(k)), k, v)
    return k, zeroed


def check_values(c, s, odd, k, zeroed, prefill):
    q, pos = rows_of(c, s)
    want, A, B, V = R.attend(q, k, zeroed, pos, c.scale)
    tol = R.bound(want, A, B, V, len(k), c.D, c.act, c.cache, prefill)
    grp = c.H // c.hk
    with np.errstate(invalid="ignore"):
        for (j, g, d), x in {o[:3]: o[3] for o in odd}.items():  # (weights are above 0 in 64 bits, and in f32 for rows like these)
            want[pos >= j, g * grp:(g + 1) * grp, d] += x
    compare(got_of(c, s), want, tol)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,lens", [(8, 2, 128, [5000, 1235]), (4, 1, 64, [9001]), (8, 8, 128, [2500, 40, 777])])
def test_decode_joins_infinite_pieces(dev, act, cache, H, hk, D, lens):
    """An infinite value in a sequence's last key: it is in the last of the pieces
    that are joined, which stands for those past it as well."""
    say("decode joins", act, cache, H, D, lens)
    c = Case(dev, seed(31, act, cache, H, D), act, cache, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens),
             decode=True)
    odds = [[(n - 1, 0, 4, np.inf), (n - 1, hk - 1, D - 3, -np.inf)] for n in lens]
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    c.run()
    for s, odd in enumerate(odds):
        check_values(c, s, odd, *plain[s], False)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", PREFILL)
def test_prefill_single_values_that_are_no_numbers(dev, act, cache, H, hk, D, past, new):
    """Single infinite and NaN elements of V, in even and odd dims, in early keys
    that all rows see, on the diagonal and behind it."""
    say("prefill single values", act, cache, H, D, past)
    c = Case(dev, seed(30, act, cache, H, D), act, cache, H, hk, D, 16, past, new, row0=1, tail=2, pad=8)
    inf, nan, g = np.inf, np.nan, hk - 1
    odds = []
    for s, (p, n) in enumerate(zip(past, new)):
        at = p + n // 2
        odds.append([(0, 0, 0, inf), (p + min(17, n - 1), g, 3, -inf), (at, 0, 6, nan), (at + 1, 0, 7, inf), (at + 1, g, 10, -inf),
                     (at + 2, 0, 7, -inf), (p + n - 1, g, D - 1, inf), (p + max(0, n - 20), 0, D - 2, nan)])
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    for _ in range(2):
        c.run()
        for s, odd in enumerate(odds):
            check_values(c, s, odd, *plain[s], True)


# 16-row tiles: cut over the workgroups, whole, a wavefront each
DECODE = [(8, 2, 128, [1500, 1235, 0, 40]), (4, 1, 64, [9001]), (8, 8, 128, [300, 1, 77, 130]), (6, 2, 64, [1] * 3 + [500]),
          (40, 20, 128, [20, 31, 2]), (64, 32, 64, [100] * 9 + [250] * 8)]


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,lens", DECODE)
def test_decode_single_values_that_are_no_numbers(dev, act, cache, H, hk, D, lens):
    """Single infinite and NaN elements of V early and late in a sequence: infinite
    where the definition is, whichever block of keys holds them."""
    say("decode single values", act, cache, H, D, lens[:4])
    c = Case(dev, seed(32, act, cache, H, D), act, cache, H, hk, D, 16, [n - 1 for n in lens], [1] * len(lens), pad=8,
             decode=True)
    inf, nan = np.inf, np.nan
    odds = [[(j, g % hk, d, x) for j, g, d, x in [(0, 0, 0, inf), (n // 3, 1, 3, -inf), (n // 2, 0, 8, nan), (n // 2, 0, 9, inf),
                                                  (n // 3, 0, 9, -inf), (n - 1, 1, D - 1, inf)]] if n else [] for n in lens]
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    for _ in range(2):
        c.run()
        for s, odd in enumerate(odds):
            check_values(c, s, odd, *plain[s], False)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new,decode", [(*x, False) for x in PREFILL] +
                         [(H, hk, D, [n - 1 for n in lens if n > 3], [1] * sum(n > 3 for n in lens), True)
                          for H, hk, D, lens in DECODE])
def test_keys_of_infinite_dims(dev, act, cache, H, hk, D, past, new, decode):
    """A key of -inf in one dim: a weight of 0 for the rows whose q is above 0
    there, no number for those below."""
    say("infinite keys", act, cache, H, D, past[:3])
    c = Case(dev, seed(33, act, cache, H, D), act, cache, H, hk, D, 16, past, new, decode=decode)
    keys = [min(2 + p + n // 2, p + n - 1) for p, n in zip(past, new)]
    plain = []
    for s, j in enumerate(keys):
        k, v = c.pool.get(s, int(c.kv[s]))
        plain.append((np.delete(k, j, 0), np.delete(v, j, 0)))
        k = k.copy()
        k[j, :, 5] = -np.inf
        c.pool.put(s, np.arange(len(k)), k, v)
    c.upload()
    c.run()
    for s, j in enumerate(keys):
        q, pos = rows_of(c, s)
        assert (q[..., 5] != 0).all() and j > 0
        want, A, B, V = R.attend(q, *plain[s], pos - (pos >= j), c.scale)
        tol = R.bound(want, A, B, V, int(c.kv[s]), D, act, cache, not decode)
        want[(pos >= j)[:, None] & (q[..., 5] < 0)] = np.nan
        compare(got_of(c, s), want, tol)
