"""Paged attention of scores so large that f32 has steps of 1 and more there: keys
whose scores are equal weigh the same, in whichever tile, walk or piece of a row they
are, over 16-bit and 8-bit caches.

Every q is 2^12 in its first dim and 0 elsewhere, every key 2^12 in that dim, so that all
products are exact and all scores are the same number: the results are the means of
the values that a row sees, with the bounds of paged_ref.py and paged8_ref.py for A = 0
(nothing is lost where equal scores are subtracted)."""
import numpy as np
import pytest

import paged8_ref as P
import paged_ref as R
import test_gpu_paged as W
import test_gpu_paged8 as W8
from paged_ref import BF16, F16, F32
from test_gpu_paged import say, seed

pytestmark = pytest.mark.gpu

TYPES = [(F32, F16), (F16, F16), (F32, BF16), (BF16, BF16), (F32, 8), (F16, 8), (BF16, 8)]
POWERS = [20, 24, 25, 26, 27, 28, 29, 31, 90]  # of the scores, in natural units


def case(dev, rng, act, cache, H, hk, D, past, new, decode):
    """A case of equal keys: keys, then values, of each sequence."""
    if cache == 8:
        c = W8.Case(dev, rng, act, H, hk, D, 16, past, new, decode=decode, fill=False)
    else:
        c = W.Case(dev, rng, act, cache, H, hk, D, 16, past, new, decode=decode)
    for s, n in enumerate(c.kv):
        k, v = np.zeros((n, hk, D), np.float32), rng.standard_normal((n, hk, D)).astype(np.float32)
        k[:, :, 0] = 2.0 ** 12
        if cache == 8:
            c.pool.append(s, 0, k, v)
        else:
            c.pool.put(s, np.arange(n), k, v)
    c.q[:] = 0
    c.q[:, ::D] = 2.0 ** 12
    return c


def means(c, s):
    """The means of what each row of sequence s sees, their bounds, and the rows' positions."""
    n, D = c.new[s], c.D
    _, v = c.pool.get(s, int(c.kv[s]))
    pos = int(c.kv[s]) - n + np.arange(n)
    want, A, B, V = R.attend(np.zeros((n, c.H, D)), np.zeros_like(v), np.nan_to_num(v), pos, 1.0)
    keys = int(c.kv[s])
    if isinstance(c, W8.Case):
        tol = P.bound(want, A, B, V, keys, D, c.act, not c.decode)
    else:
        tol = R.bound(want, A, B, V, keys, D, c.act, c.cache, not c.decode)
    return want, tol, pos


# decode cut; 16-row tiles whole; 128-row tiles
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", [
    (4, 2, 128, [2299, 39], [1, 1]), (4, 2, 128, [60, 0], [9, 30]), (20, 20, 64, [0, 3] * 7, [130, 71] * 7)])
def test_equal_scores(dev, act, cache, H, hk, D, past, new):
    rng = seed(50, act, cache, H, D)
    c = case(dev, rng, act, cache, H, hk, D, past, new, new[0] == 1)
    c.upload()
    exact = [means(c, s) for s in range(len(new))]
    for power in POWERS:
        say("equal scores", act, cache, H, D, past, power)
        c.run(2.0 ** (power - 24))
        out = c.got()
        for s, (want, tol, _) in enumerate(exact):
            got = out[c.start[s]:c.start[s] + c.new[s], :H * D].reshape(want.shape)
            bad = np.argwhere(~(np.abs(got - want) <= tol))
            assert not len(bad), (power, s, bad[:3], got[tuple(bad[0])], want[tuple(bad[0])])


# 64-row tiles, the keys of a tile in two halves; cut 128-row tiles
@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", [
    (20, 20, 64, [0, 70, 0], [330, 260, 130]), (32, 2, 128, [0, 30], [170, 60]),
    (32, 2, 128, [2200, 2000, 0], [150, 100, 40]), (40, 2, 64, [2200, 2000], [150, 140])])
def test_equal_scores_in_pieces(dev, act, cache, H, hk, D, past, new):
    """Pieces of few and of many keys: each counts by its keys."""
    test_equal_scores(dev, act, cache, H, hk, D, past, new)


@pytest.mark.parametrize("act,cache", TYPES)
@pytest.mark.parametrize("H,hk,D,past,new", [
    (4, 2, 128, [60, 0], [9, 30]), (20, 20, 64, [0, 3] * 7, [130, 71] * 7), (20, 20, 64, [0, 70, 0], [330, 260, 130]),
    (32, 2, 128, [2200, 2000, 0], [150, 100, 40])])
def test_equal_scores_beside_nan(dev, act, cache, H, hk, D, past, new):
    """A NaN in one dim of a value that the later half of a sequence's rows see: its tile's keys are
    taken one after another, and weigh as those of the others do."""
    rng = seed(51, act, cache, H, D)
    c = case(dev, rng, act, cache, H, hk, D, past, new, False)
    at = [int(k) - n // 2 for k, n in zip(c.kv, new)]
    for s, j in enumerate(at):
        page, i = c.pool.table[s, j // 16], j % 16
        if cache == 8:
            c.pool.code[1, page, :, i, 1] = P.NAN
        else:
            c.pool.v[page, :, i, 1] = R.NAN[cache]
    c.upload()
    exact = [means(c, s) for s in range(len(new))]
    for power in POWERS:
        say("equal scores beside NaN", act, cache, H, D, past, power)
        c.run(2.0 ** (power - 24))
        out = c.got()
        for s, (want, tol, pos) in enumerate(exact):
            got = out[c.start[s]:c.start[s] + c.new[s], :H * D].reshape(want.shape)
            nan = np.zeros(want.shape, bool)
            nan[pos >= at[s], :, 1] = True
            np.testing.assert_array_equal(np.isnan(got), nan)
            bad = np.argwhere(~nan & ~(np.abs(got - want) <= tol))
            assert not len(bad), (power, s, bad[:3], got[tuple(bad[0])], want[tuple(bad[0])])
