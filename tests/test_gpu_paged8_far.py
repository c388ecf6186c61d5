"""8-bit paged attention of values whose scales lie far apart, and of codes that stand for
more than f32 holds: what rows of every type make of them, and what such a batch costs
beside one of scales that are alike."""
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
@pytest.mark.parametrize("low,high", [(-60, 12), (-20, 5), (-8, 60), (110, 120), (-80, -60)])
def test_values_far_apart(dev, act, H, hk, D, past, new, low, high):
    """Every block of values 2^low .. 2^high in size, some of zeros: within f16's range, within
    what f16 holds of the largest, past f16's range, near f32's end, below f16's least."""
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


BIG = float(np.finfo(np.float32).max)
# (position from the end, scale byte, code, dim): infinite from 2^128 on
PAST = [(5, 254, 0x7e, 3), (5, 254, 0x01, 4), (40, 247, 0x78, 5), (40, 247, 0x77, 6), (41, 247, 0xf8, 7), (70, 250, 0xfe, 8),
        (70, 250, 0x58, 9), (71, 250, 0x3f, 10), (100, 246, 0x7e, 11), (5, 254, 0xb1, 12), (41, 247, 0xf8, 3)]


def plant(c, s, w):
    """PAST in k (0) or v (1) of sequence s, their blocks zeros beside them."""
    n, done = int(c.kv[s]), set()
    for back, b, code, d in PAST:
        j = n - back
        if j < 0:
            continue
        page, i = c.pool.table[s, j // 16], j % 16
        if j // 16 not in done:
            c.pool.code[w, page] = 0
            c.pool.scale[w, page] = b
            done.add(j // 16)
        if c.pool.scale[w, page, 0, 0] == b:
            c.pool.code[w, page, :, i, d] = code


def in_f32(x):
    return np.where(np.abs(x) > BIG, np.copysign(np.inf, x), x)


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", KINDS + [(4, 2, 128, [599, 2300], [1, 1]), (4, 2, 64, [599, 80], [1, 1])])
@pytest.mark.parametrize("power", [0, 118])
def test_values_past_f32(dev, act, H, hk, D, past, new, power):
    """Infinite where a code times its scale is, for the rows that see it, beside values of
    2^power."""
    say("values past f32", act, H, D, past, power)
    rng = seed(62, act, H, D)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, decode=new == [1, 1], fill=False)
    for s, n in enumerate(c.kv):
        k, v = rng.standard_normal((2, n, hk, D)).astype(np.float32)
        c.pool.append(s, 0, k, v * np.float32(2.0 ** power))
        plant(c, s, 1)
    c.upload()
    c.run()
    for s, n in enumerate(new):
        r0, kv = int(c.start[s]), int(c.kv[s])
        k, v = c.pool.get(s, kv)
        v = in_f32(v)
        pos = kv - n + np.arange(n)
        q = R.from_bits(R.to_bits(c.q, act), act)[r0:r0 + n, :H * D].reshape(n, H, D)
        inf = np.isinf(v)
        want, A, B, _ = R.attend(q, k, np.where(inf, 0, v), pos, c.scale)
        V = np.maximum.accumulate(np.abs(np.where(inf, 0, v)).max((1, 2)))[pos][:, None, None]
        tol = P.bound(want, A, B, V, kv, D, act, not c.decode)
        with np.errstate(invalid="ignore"):
            for j, g, d in np.argwhere(inf):
                want[pos >= j, g * H // hk:(g + 1) * H // hk, d] += v[j, g, d]
        got = c.got()[r0:r0 + n, :H * D].reshape(want.shape)
        most = 65520.0 if act == F16 else BIG
        with np.errstate(invalid="ignore"):
            past_it = np.abs(want) - tol > most  # (f16 holds no more; infinities)
            near = ~past_it & (np.abs(want) + tol > most)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        np.testing.assert_array_equal(got[past_it], np.where(want[past_it] > 0, np.inf, -np.inf))
        fine = ~past_it & ~near & ~np.isnan(want)
        bad = np.argwhere(~(np.abs(got[fine] - want[fine]) <= tol[fine]))
        assert not len(bad), (s, np.argwhere(fine)[bad[:3, 0]], len(bad))


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", KINDS + [(4, 2, 128, [599, 2300], [1, 1]), (4, 2, 64, [599, 80], [1, 1])])
def test_keys_past_f32(dev, act, H, hk, D, past, new):
    """Infinite keys: no weight where q is below zero in their infinite dim, NaN for rows that see
    one and are above zero or zero there."""
    say("keys past f32", act, H, D, past)
    rng = seed(63, act, H, D)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, decode=new == [1, 1])
    c.q = c.q.reshape(c.rows, H, D)
    sign = np.where(np.arange(H) % 3 < 2, -1.0, np.where(np.arange(H) % 2, 0.0, 1.0)).astype(np.float32)
    c.q[:, :, 3:13] = sign[:, None] * (np.abs(c.q[:, :, 3:13]) + 0.25)
    c.q = c.q.reshape(c.rows, H * D)
    ats = [(5, 3, 0x7e), (40, 5, 0x78), (70, 8, 0x7e)]  # each an infinity above zero
    for s in range(len(new)):
        for back, d, code in ats:
            j = int(c.kv[s]) - back
            if j < 0:
                continue
            page, i = c.pool.table[s, j // 16], j % 16
            c.pool.code[0, page] = 0
            c.pool.scale[0, page] = 254 if back == 5 else 247 if back == 40 else 251
            c.pool.code[0, page, :, i, d] = code
    c.upload()
    c.run()
    for s, n in enumerate(new):
        r0, kv = int(c.start[s]), int(c.kv[s])
        k, v = c.pool.get(s, kv)
        inf = (np.abs(k) > BIG).any((1, 2))
        left = np.flatnonzero(~inf)
        pos = kv - n + np.arange(n)
        q = R.from_bits(R.to_bits(c.q, act), act)[r0:r0 + n].reshape(n, H, D)
        at = np.searchsorted(left, pos, side="right") - 1  # the last of those left that a row sees
        want, A, B, V = R.attend(q, k[left], v[left], at, c.scale)
        tol = P.bound(want, A, B, V, kv, D, act, not c.decode)
        sees = (np.flatnonzero(inf)[None] <= pos[:, None]).any(1)
        got = c.got()[r0:r0 + n].reshape(want.shape)
        nan = sees[:, None] & ((sign >= 0)[None] | (at < 0)[:, None])  # (scores of -inf alone: 0 / 0)
        np.testing.assert_array_equal(np.isnan(got).all(2), nan)
        bad = np.argwhere(~nan[..., None] & ~(np.abs(got - want) <= tol))
        assert not len(bad), (s, bad[:3], len(bad))


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", KINDS + [(4, 2, 128, [599, 2300], [1, 1])])
def test_values_of_2_to_the_minus_100(dev, act, H, hk, D, past, new):
    """Weights are 2^-31 at most where V is taken as values, 2^-38 or more of a row's largest: each
    product may lose a step of f32's least, 2^-149, which is 2^-111 of the result."""
    say("tiny values", act, H, D, past)
    rng = seed(64, act, H, D)
    c = Case(dev, rng, act, H, hk, D, 16, past, new, decode=new == [1, 1], fill=False)
    for s, n in enumerate(c.kv):
        k, v = rng.standard_normal((2, n, hk, D)).astype(np.float32)
        c.pool.append(s, 0, k, v * np.float32(2.0 ** -100))
    c.upload()
    c.run()
    for s, n in enumerate(new):
        r0, kv = int(c.start[s]), int(c.kv[s])
        k, v = c.pool.get(s, kv)
        pos = kv - n + np.arange(n)
        q = R.from_bits(R.to_bits(c.q, act), act)[r0:r0 + n, :H * D].reshape(n, H, D)
        want, A, B, V = R.attend(q, k, v, pos, c.scale)
        tol = P.bound(want, A, B, V, kv, D, act, not c.decode) + kv * 2.0 ** -111
        got = c.got()[r0:r0 + n, :H * D].reshape(want.shape)
        assert (np.abs(got - want) <= tol).all()
