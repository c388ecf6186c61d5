"""Appends to an 8-bit paged KV cache at the ends of its scales: graded finite values up to
f32's largest under the last scale, on their own and beside older rows, and older rows
whose block's scale grows."""
import numpy as np
import pytest

import fuel_amd as F
import paged8_ref as P
from paged_ref import F32
from test_gpu_paged8 import Case, put, say, seed

pytestmark = pytest.mark.gpu

BIG = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_append_up_to_the_largest_number(dev, one, D):
    """The last scale is 2^120: codes up to 240 stand for numbers of f32 there."""
    say("append to the end", one, D)
    e = np.arange(D)
    blocks = [np.linspace(-BIG, BIG, D), BIG * 2.0 ** -(e / 3.0), np.linspace(BIG * 0.8, BIG, D) * (-1.0) ** e,
              np.r_[np.full(D - 1, 448.0 * 2.0 ** 119), 240.0 * 2.0 ** 120], np.r_[np.full(D - 1, 1.0), BIG],
              np.r_[240.0, 244.0, 247.9, 248.0, 252.0, -248.0, np.zeros(D - 6)] * 2.0 ** 120,
              np.r_[448.0, 449.0, np.zeros(D - 2)] * 2.0 ** 119, np.r_[448.0, np.zeros(D - 1)] * 2.0 ** 119]
    x = np.asarray(blocks, np.float32)
    assert np.isfinite(x).all()
    n = len(x)
    past = [0] * n + [3] * n + [16] * n + [15] * n
    c = Case(dev, seed(70, D), F32, 1, 1, D, 16, past, [1] * 4 * n, decode=one, fill=False)
    for s, p in enumerate(past):
        c.pool.fill(seed(71, s), s, p, std=[1.0, 2.0 ** 118, 2.0 ** 100][s % 3])
    x = np.concatenate([x] * 4)
    c.upload()
    xd, yd = put(dev, x), put(dev, -x)
    F.paged_append(c.kvc, c.batch, F32, 1, None, xd, yd, None)
    for s, p in enumerate(past):
        c.pool.append(s, p, x[s].reshape(1, 1, D), -x[s].reshape(1, 1, D))
    c.check_cells()
    for s in range(4 * n):
        k, v = c.pool.get(s, int(c.kv[s]))
        assert (np.abs(k) < 2.0 ** 128).all() and (np.abs(v) < 2.0 ** 128).all()
    assert c.pool.scale.max() <= 255 and (c.pool.scale == 247).any() and (c.pool.scale == 246).any()


@pytest.mark.parametrize("one", [False, True])
def test_older_rows_under_a_grown_scale(dev, one):
    """Exact from 2^-6 in units of the new scale on, 2^-13.8 of the block's largest; below, the
    nearest multiple of 2^-9."""
    say("grown scale", one)
    D = 64
    old = np.zeros((3, 1, D), np.float32)
    old[:, 0, :] = 2.0 ** -5 * (1 + np.arange(D) % 8 / 8) * 2.0 ** (np.arange(D) // 8 - 3)[None]  # from 2^-8 on
    tops = [450.0, 896.0, 897.0, 448.0, 2.0 ** 20, 30.0]
    c = Case(dev, seed(72), F32, 1, 1, D, 16, [3] * len(tops), [1] * len(tops), decode=one, fill=False)
    old[0, 0, 0] = 448.0  # byte 127
    for s in range(len(tops)):
        c.pool.append(s, 0, old, old)
    before = c.pool.get(0, 3)[0]
    c.upload()
    x = np.zeros((len(tops), D), np.float32)
    x[:, 1] = tops
    xd = put(dev, x)
    F.paged_append(c.kvc, c.batch, F32, 1, None, xd, xd, None)
    lost = 0
    for s, top in enumerate(tops):
        c.pool.append(s, 3, x[s].reshape(1, 1, D), x[s].reshape(1, 1, D))
        after = c.pool.get(s, 3)[0]
        unit = P.scale(int(P.byte(max(top, 448.0))))
        keeps = np.abs(before) >= 2.0 ** -6 * unit
        np.testing.assert_array_equal(after[keeps], before[keeps])
        assert (np.abs(after - before) <= 2.0 ** -10 * unit).all()
        assert (np.abs(before[after != before]) < 2.0 ** -13.8 * max(top, 448.0)).all()
        lost += (after != before).sum()
    assert lost > 0
    c.check_cells()
