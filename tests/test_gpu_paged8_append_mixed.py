"""Appends of batches that mix sequences of no, of few and of many rows to an 8-bit paged
KV cache, as padded batches of a server do: bit-exact, and at the cost of their rows."""
import time

import numpy as np
import pytest

import fuel_amd as F
import paged_ref as R
from paged_ref import BF16, F16, F32
from test_gpu_paged8 import TYPES, Case, put, say, seed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", TYPES)
@pytest.mark.parametrize("hk,D,ps", [(1, 64, 16), (9, 128, 32), (20, 64, 64)])
@pytest.mark.parametrize("idle", [40, 300])
def test_append_of_few_and_of_many_rows(dev, act, hk, D, ps, idle):
    """Sequences of 0 .. 8 rows from every position of a block on, longer ones beside them, a
    length that is none, a page that is none, rows before position 0 and past the tables."""
    say("append mixed", act, hk, D, idle)
    rng = seed(80, act, hk, idle)
    new = [n for n in range(1, 9) for _ in range(4)] + [16, 17, 31, 40, 5, 4, 4, 6, 3, 7] + [0] * idle
    past = [int(x) for x in rng.integers(0, 34, len(new))]
    past[-idle - 4], past[-idle - 3] = -2, -2  # of 4 and 6 rows
    order = rng.permutation(len(new))
    new, past = [new[i] for i in order], [max(past[i], -new[i]) for i in order]
    c = Case(dev, rng, act, hk, hk, D, ps, past, new, tail=2, fill=False, width=5 if ps == 16 else 0)
    assert (c.rows <= 2 * len(new)) == (idle == 300)
    for s, p in enumerate(past):
        c.pool.fill(rng, s, p, std=[1.0, 2.0 ** -9, 2.0 ** 9][s % 3])
    threes = [s for s, n in enumerate(new) if n == 3 and past[s] > 0]
    c.kv[threes[0]] = c.pool.table.shape[1] * ps + 1
    c.pool.table[threes[1], past[threes[1]] // ps] = -1
    cos, sin = R.tables(36, D)
    c.upload()
    k, v = rng.standard_normal((2, c.rows, hk * D)).astype(np.float32)
    k *= (2.0 ** rng.integers(-9, 9, c.rows)).astype(np.float32)[:, None]
    kd, vd, qd = put(dev, k, act), put(dev, v, act), put(dev, k, act)
    qo = put(dev, np.full((c.rows, hk * D), 7.0), act)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    F.paged_append(c.kvc, c.batch, act, hk, qd, kd, vd, qo, rope_cos=cd, rope_sin=sd, rope_rows=36)
    k, v = (R.from_bits(R.to_bits(a, act), act).reshape(c.rows, hk, D) for a in (k, v))
    want = np.full((c.rows, hk * D), 7.0, np.float32)
    for s, n in enumerate(new):
        if not n:
            continue
        r = slice(c.start[s], c.start[s] + n)
        pos = int(c.kv[s]) - n + np.arange(n)
        turned = R.rotate(k[r], cos[np.clip(pos, 0, 35)], sin[np.clip(pos, 0, 35)])
        on = (pos >= 0) & (pos < 36)
        q = np.where((pos < 0)[:, None, None], 0, turned)
        q[pos >= 36] = np.nan
        if s == threes[0]:
            q[:], on[:] = np.nan, False
        want[r] = q.reshape(n, -1)
        if on.any():
            c.pool.append(s, int(pos[on][0]), turned[on], v[r][on])
    got = qo.numpy()
    np.testing.assert_array_equal(np.isnan(R.from_bits(got, act)), np.isnan(want))
    ok = ~np.isnan(want)
    np.testing.assert_array_equal(got[ok], R.to_bits(want, act)[ok])
    c.check_cells()


@pytest.mark.parametrize("hk", [8, 32])
def test_one_prompt_among_idle_slots(dev, hk):
    """1000 rows of one sequence beside 511 empty ones, and alone: below three times the time (it
    was six: a wavefront took a block's rows one after another)."""
    say("one prompt", hk)
    times = []
    for slots in (1, 512):
        c = Case(dev, seed(81), BF16, hk, hk, 128, 16, [0] * slots, [0] * (slots - 1) + [1000], fill=False)
        c.upload()
        k = put(dev, np.zeros((c.rows, hk * 128)), BF16)
        best = np.inf
        for _ in range(8):
            t = time.perf_counter()
            for _ in range(20):
                F.paged_append(c.kvc, c.batch, BF16, hk, None, k, k, None)
            dev.synchronize()
            best = min(best, (time.perf_counter() - t) / 20)
        times.append(best)
    say("   us", [round(1e6 * t, 1) for t in times])
    assert times[1] < 3 * times[0]
