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


# heads, KV heads, dims, cached, new: 64-row tiles, 128-row tiles, cut 128-row tiles
PREFILL = [(32, 2, 128, [0, 30], [170, 160]), (64, 4, 64, [0, 30], [170, 160]), (20, 20, 128, [0, 0, 70, 0, 3], [200, 260, 130, 60, 200]),
           (40, 20, 64, [0, 0, 70], [200, 260, 130]), (32, 2, 128, [2200, 2000], [150, 140]),
           (40, 2, 64, [2200, 2000], [150, 140])]


def put_values(c, s, odd):
    """odd: (key, KV head, dim, value) of sequence s's V; its keys, and V with zeros there."""
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
        for j, g, d, x in odd:  # (weights are above 0 in 64 bits, and in f32 for rows like these)
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
        odds.append([(0, 0, 0, inf), (p + 17, g, 3, -inf), (at, 0, 6, nan), (at + 1, 0, 7, inf), (at + 1, g, 10, -inf),
                     (at + 2, 0, 7, -inf), (p + n - 1, g, D - 1, inf), (p + n - 20, 0, D - 2, nan)])
    plain = [put_values(c, s, odd) for s, odd in enumerate(odds)]
    c.upload()
    for _ in range(2):
        c.run()
        for s, odd in enumerate(odds):
            check_values(c, s, odd, *plain[s], True)
