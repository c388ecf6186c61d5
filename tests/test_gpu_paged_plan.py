"""Pages of a pool for the sequences of a batch (frq_paged_plan) against the rules
sequence by sequence, and the operators of a server's step together: plan, append,
attention, captured and replayed while sequences come, grow and end."""
import numpy as np
import pytest

import fuel_amd as F
import paged8_ref as P
import paged_ref as R
from fuel_amd.hiprt import HipRuntime
from paged_ref import BF16, F32
from test_gpu_paged8 import put, say, seed

pytestmark = pytest.mark.gpu


def plan(tokens, kv, table, free, n_free, ps, rows):
    """The rules, one sequence after the other: everything a call writes."""
    n, width = table.shape
    kv, table, free = [int(x) for x in kv], table.copy(), free.copy()
    have, cap = min(max(int(n_free), 0), len(free)), width * ps
    t = [int(x) if 0 <= k <= cap and x <= cap - k else 0 for x, k in zip(tokens, kv)]
    up = lambda x: -(-x // ps)  # noqa: E731
    for s in range(n):
        if t[s] < 0:
            end = max(0, kv[s] + t[s])
            for i in range(up(end), up(kv[s])):
                if have < len(free):
                    free[have] = table[s, i]
                    have += 1
            kv[s] = end
    top, pages, asked, start, slots, pos = have, 0, 0, [0], [], []
    for s in range(n):
        if t[s] > 0:
            a, b = up(kv[s]), up(kv[s] + t[s])
            pages, asked = pages + b - a, asked + t[s]
            if (a == b or pages <= top) and asked <= rows:
                for i in range(a, b):
                    have -= 1
                    table[s, i] = free[have]
                for j in range(kv[s], kv[s] + t[s]):
                    slots.append(int(table[s, j // ps]) * ps + j % ps)
                    pos.append(j)
                kv[s] += t[s]
        start.append(len(slots))
    pad = [-1] * (rows - len(slots))
    return np.array(kv), table, free, have, np.array(start), np.array(slots + pad), np.array(pos + pad)


class Call:
    def __init__(self, dev, tokens, kv, table, free, n_free, ps, rows):
        self.want = plan(tokens, kv, table, free, n_free, ps, rows)
        self.n, self.width, self.ps, self.rows, self.n_pages = *table.shape, ps, rows, len(free)
        i = lambda a, t=np.int32: dev.from_numpy(np.asarray(a, t))  # noqa: E731
        self.dev = dev
        self.tokens, self.kv, self.table, self.free, self.n_free = map(i, (tokens, kv, table, free, [n_free]))
        self.kv_out, self.n_out = i(np.full(self.n, 77)), i([77])
        self.start = i(np.full(self.n + 1, 77))
        self.slots, self.pos = i(np.full(rows, 77), np.int64), i(np.full(rows, 77))

    def run(self, apart=True, slots=True, positions=True):
        F.paged_plan(self.dev, self.n, self.width, self.ps, self.n_pages, self.rows, self.tokens, self.kv, self.table,
                     self.free, self.n_free, self.start, self.slots if slots else None,
                     self.pos if positions else None, *((self.kv_out, self.n_out) if apart else ()))
        got = (self.kv_out if apart else self.kv, self.table, self.free, self.n_out if apart else self.n_free,
               self.start, self.slots, self.pos)
        for name, x, w, on in zip(("kv_len", "page_table", "free_pages", "n_free", "row_start", "slots", "positions"),
                                  got, self.want, (1, 1, 1, 1, 1, slots, positions)):
            np.testing.assert_array_equal(x.numpy().reshape(np.shape(w)), w if on else np.full(np.shape(w), 77), name)


def batch(rng, n, ps, width, new, share=1.0, ended=5):
    cap = width * ps
    kv = rng.integers(0, cap + 1, n)
    up = -(-kv // ps)
    table = np.full((n, width), 1 << 29, np.int32)
    asked = int(sum(-(-min(cap, k + new) // ps) - u for k, u in zip(kv, up)))
    order = rng.permutation(int(up.sum()) + int(asked * share) + 1)
    at = 0
    for s in range(n):
        table[s, :up[s]] = order[at:at + up[s]]
        at += up[s]
    free = np.zeros(len(order), np.int32)
    free[:len(order) - at] = order[at:]
    tokens = rng.integers(0, new + 1, n)
    tokens[::ended] = -rng.integers(0, cap + 40, len(tokens[::ended]))
    return tokens, kv, table, free, len(order) - at, ps


@pytest.mark.parametrize("n,ps,width,new", [(1, 16, 3, 20), (7, 16, 9, 40), (64, 32, 5, 1), (300, 16, 20, 200),
                                            (1023, 64, 3, 5), (1024, 16, 4, 30), (1025, 16, 4, 30), (5000, 128, 2, 3)])
@pytest.mark.parametrize("share", [1.2, 0.5, 0.0])
def test_plan(dev, n, ps, width, new, share):
    say("plan", n, ps, width, new, share)
    rng = seed(60, n, width, int(10 * share))
    b = batch(rng, n, ps, width, new, share)
    most = int(np.maximum(b[0], 0).sum())
    for i, rows in enumerate((most + 3, max(1, most // 2))):
        Call(dev, *b, rows).run()
        Call(dev, *b, rows).run(apart=False, slots=i == 0, positions=i == 1)


def test_plan_entries_that_are_none(dev):
    """Lengths that are none, tokens past every range, a stack of more pages than there
    are or of fewer than none, more dropped than the stack holds."""
    say("plan malformed")
    rng = seed(61)
    lo, hi = -(1 << 31), (1 << 31) - 1
    tokens, kv, table, free, n_free, ps = batch(rng, 40, 16, 6, 50)
    kv[:6] = -1, lo, hi, 97, 96, 96
    tokens[:6] = 5, -5, 1, 1, 1, hi
    tokens[6:12] = lo, hi, -1, 1 << 30, lo + 1, -97
    for have in (n_free, 0, -5, lo, hi, len(free), len(free) - 1):
        for rows in (0, 1, 300):
            c = Call(dev, tokens, kv, table, free, have, ps, rows)
            c.run(slots=rows > 0, positions=rows > 0)
    # every sequence drops more pages than the pool has, over and over
    n = 3000
    c = Call(dev, np.full(n, lo), np.full(n, 1 << 10), np.arange(n * 64).reshape(n, 64) % 50, np.zeros(50, np.int32),
             3, 16, 4)
    c.run()


@pytest.mark.parametrize("n,ps,width", [(6, 1024, 1 << 20), (1100, 1024, 1 << 11), (1100, 16, 1 << 14)])
def test_plan_sums_past_32_bits(dev, n, ps, width):
    """More tokens and pages asked for than an int counts, small requests between."""
    say("plan sums", n, ps, width)
    rng = seed(63, n, ps)
    cap = width * ps
    for pages, rows in ((40, 2000), (3, 2000), (40, 7), (1000, 1 << 12)):
        kv = rng.integers(0, 3, n)
        table = np.full((n, width), -1, np.int32)
        table[:, 0] = 1000 + np.arange(n)
        tokens = rng.integers(0, 20, n)
        tokens[rng.integers(0, n, n // 2)] = cap - 3
        tokens[0], tokens[1], tokens[-1] = 2, 3, -1
        Call(dev, tokens, kv, table, np.arange(pages), pages, ps, rows).run()


def test_plan_of_nothing(dev):
    say("plan of nothing")
    i = lambda a, t=np.int32: dev.from_numpy(np.asarray(a, t))  # noqa: E731
    start, n_free, slots = i([9]), i([2]), i([9, 9], np.int64)
    F.paged_plan(dev, 0, 4, 16, 3, 2, None, None, None, i([0, 1, 2]), n_free, start, slots)
    assert start.numpy()[0] == 0 and n_free.numpy()[0] == 2 and (slots.numpy() == -1).all()


@pytest.mark.parametrize("act,H,hk,D", [(F32, 4, 2, 128), (BF16, 8, 1, 64)])
def test_a_server_of_captured_steps(dev, act, H, hk, D):
    """Sequences that come with prompts, grow by a token a step and end: a step is one
    recording of plan, append and attention over an 8-bit cache, replayed with other
    tokens, the pool too small for all at once, eager work between.  Every row's
    output against attention over what its sequence has appended so far."""
    rng = seed(62, act)
    say("a server", act)
    n, width, ps, n_pages, rows = 6, 8, 16, 11, 90
    w = (H + 2 * hk) * D
    cos, sin = R.tables(width * ps, D)
    cd, sd = dev.from_numpy(cos), dev.from_numpy(sin)
    kvc = F.PagedKvCache8(dev, n_pages, ps, hk, D)
    i = lambda a, t=np.int32: dev.from_numpy(np.asarray(a, t))  # noqa: E731
    order = rng.permutation(n_pages)
    tokens, kv, table = i(np.zeros(n)), i(np.zeros(n)), i(np.full((n, width), -1))
    free, n_free, start = i(order), i([n_pages]), i(np.zeros(n + 1))
    slots, pos = i(np.zeros(rows), np.int64), i(np.zeros(rows))
    b = F.PagedBatch(table, kv, n, width, rows, start)
    work = dev.alloc((max(16, F.paged_attention_workspace(kvc, b, H)),), np.uint8)
    scale = float(np.float32(D ** -0.5))
    x = put(dev, np.zeros((rows, w)), act)
    size = x.nbytes // rows // w
    qd, od = put(dev, np.zeros((rows, H * D)), act), put(dev, np.zeros((rows, H * D)), act)

    def step():
        F.paged_plan(dev, n, width, ps, n_pages, rows, tokens, kv, table, free, n_free, start, slots, pos)
        F.paged_append(kvc, b, act, H, x, x.ptr + H * D * size, x.ptr + (H + hk) * D * size, qd, ldq=w, ldk=w, ldv=w,
                       rope_cos=cd, rope_sin=sd, rope_rows=width * ps)
        F.paged_attention_prefill(kvc, b, act, H, qd, od, scale, work)

    state = [np.zeros(n, np.int64), np.full((n, width), -1, np.int32), order.astype(np.int32), n_pages]
    pool = P.Pool(rng, [0], ps, hk, D, spare=n_pages)
    pool.code[:], pool.scale[:] = 0, 0
    rt = HipRuntime()
    stream = rt.stream_create()
    dev.synchronize()
    dev.set_stream(stream)
    refused = 0
    try:
        graph = rt.capture(stream, step)
        for t in range(30):
            ask = np.where(state[0] == 0, rng.integers(0, 2, n) * rng.integers(1, 60, n), 1)
            ask[(state[0] > 0) & (rng.random(n) < 0.12)] = -1000
            if t % 7 == 3:
                ask[rng.integers(0, n)] = -3
            before = state[0]
            *state, ranges, want_slots, want_pos = plan(ask, *state, ps, rows)
            refused += int(((ask > 0) & (np.diff(ranges) == 0)).sum())
            xs = rng.standard_normal((rows, w)).astype(np.float32)
            x.copy_from(R.to_bits(xs, act))
            tokens.copy_from(ask.astype(np.int32))
            if t % 4 == 2:
                step()  # eager
            else:
                rt.graph_launch(graph, stream)
            rt.stream_sync(stream)
            for got, want in zip((kv, table, free, n_free, start, slots, pos), (*state, ranges, want_slots, want_pos)):
                np.testing.assert_array_equal(got.numpy().reshape(np.shape(want)), want)
            xs = R.from_bits(R.to_bits(xs, act), act)
            out = R.from_bits(od.numpy(), act)
            pool.table = state[1]
            for s in range(n):
                lo, hi = ranges[s], ranges[s + 1]
                if lo == hi:
                    continue
                at = np.arange(state[0][s] - (hi - lo), state[0][s])
                assert at[0] == max(0, before[s] + min(ask[s], 0))
                q, k, v = (a.reshape(hi - lo, -1, D) for a in np.split(xs[lo:hi], [H * D, (H + hk) * D], 1))
                pool.append(s, int(at[0]), R.rotate(k, cos[at], sin[at]), v)
                q = R.from_bits(R.to_bits(R.rotate(q, cos[at], sin[at]), act), act)
                keys, values = pool.get(s, int(state[0][s]))
                want, A, B, V = R.attend(q, keys, values, at, scale)
                tol = P.bound(want, A, B, V, int(state[0][s]), D, act, True)
                assert (np.abs(out[lo:hi].reshape(want.shape) - want) <= tol).all(), (t, s)
        rt.graph_destroy(graph)
    finally:
        dev.set_stream(None)
        rt.stream_destroy(stream)
    assert refused  # (some did not fit)
