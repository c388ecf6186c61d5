"""8-bit paged attention of values whose scales lie far apart: what rows of every type
keep of them, and what such a batch costs beside one of scales that are alike."""
import time

import numpy as np
import pytest

import paged8_ref as P
import paged_ref as R
from paged_ref import BF16, F16, F32
from test_gpu_paged8 import TYPES, Case, say, seed

pytestmark = pytest.mark.gpu

# 16-row tiles, 64-row tiles, 128-row tiles, cut 128-row tiles
KINDS = [(4, 2, 128, [60, 0], [9, 30]), (32, 2, 128, [0, 30], [170, 60]), (20, 20, 64, [0, 3] * 7, [130, 71] * 7),
         (32, 2, 128, [2200, 2000, 0], [150, 100, 40])]


def check(c, s, most=np.inf):
    """Sequence s's rows against the definition, each value's size counted for the rows
    that see it only; results past `most` in magnitude are infinite, of the same sign."""
    n, r0, D = c.new[s], int(c.start[s]), c.D
    k, v = c.pool.get(s, int(c.kv[s]))
    pos = int(c.kv[s]) - n + np.arange(n)
    q = R.from_bits(R.to_bits(c.q, c.act), c.act)[r0:r0 + n, :c.H * D].reshape(n, c.H, D)
    want, A, B, _ = R.attend(q, k, v, pos, c.scale)
    V = np.maximum.accumulate(np.abs(v).max((1, 2)))[pos][:, None, None]
    tol = P.bound(want, A, B, V, int(c.kv[s]), D, c.act, not c.decode)
    got = c.got()[r0:r0 + n, :c.H * D].reshape(want.shape)
    past, near = np.abs(want) - tol > most, np.abs(want) + tol > most
    np.testing.assert_array_equal(got[past], np.where(want[past] > 0, np.inf, -np.inf))
    either = near & ~past  # (the bound holds numbers and infinities)
    bad = np.argwhere(~near & ~(np.abs(got - want) <= tol))
    assert not len(bad), (s, bad[:3], len(bad))
    assert not np.isnan(got).any() and either.sum() <= got.size // 50
    return past.sum()


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", KINDS + [(4, 2, 128, [599, 2300], [1, 1]), (4, 2, 64, [599, 80], [1, 1])])
@pytest.mark.parametrize("low,high", [(-60, 12), (-20, 5), (-8, 60)])
def test_values_far_apart(dev, act, H, hk, D, past, new, low, high):
    """Every block of values 2^low .. 2^high in size, some of zeros: within f16's range, within
    what f16 holds of the largest, and past f16's range."""
    say("values far apart", act, H, D, past, low, high)
    rng = seed(60, act, H, D, low + 100)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, fill=False, decode=new == [1, 1])
    for s, n in enumerate(c.kv):
        k, v = rng.standard_normal((2, n, hk, D)).astype(np.float32)
        size = rng.integers(low, high + 1, n // 16 + 1).repeat(16)[:n]
        v *= (2.0 ** size * (rng.integers(0, 8, n // 16 + 1) > 0).repeat(16)[:n])[:, None, None]
        k *= 2.0 ** rng.integers(-3, 2, n // 16 + 1).repeat(16)[:n][:, None, None]
        c.pool.append(s, 0, k.astype(np.float32), v.astype(np.float32))
    c.upload()
    c.run()
    most = 65520.0 if act == F16 else np.inf
    for s in range(len(new)):
        check(c, s, most)


@pytest.mark.parametrize("act", [F32, F16])
@pytest.mark.parametrize("H,hk,past,new", [(32, 8, [0], [4000]), (32, 32, [1306, 2169], [322, 451]),
                                           (32, 8, [8000], [512]), (32, 8, [600], [300])])
def test_scales_far_apart_cost_a_second_walk(dev, act, H, hk, past, new):
    """One block of tiny values in each head: the keys are walked twice, by matrix instructions
    both times.  (1.5 times the products of the first walk; below 6 times the call.)"""
    say("cost", act, H, hk, past)
    rng = seed(61)
    c = Case(dev, rng, act, H, hk, 128, 16, past, new, fill=False)
    c.pool.code[:] = rng.integers(0, 120, c.pool.code.shape, dtype=np.uint8)
    times = []
    for far in (False, True):
        c.pool.scale[:] = 119
        if far:
            c.pool.scale[1, c.pool.table[:, 0]] = 119 - 40
        c.upload()
        for _ in range(3):
            c.run()
        dev.synchronize()
        best = np.inf
        for _ in range(5):
            t = time.perf_counter()
            for _ in range(4):
                c.run()
            dev.synchronize()
            best = min(best, time.perf_counter() - t)
        times.append(best / 4)
    say("   us", [round(1e6 * t, 1) for t in times])
    assert times[1] < 6 * times[0]
