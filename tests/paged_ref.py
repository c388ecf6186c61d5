"""Plain 64-bit forms of the paged KV cache operators, the bounds their outputs
are held to, and the host-side pool the tests fill.

Bounds.  u = 2^-24 (half a step of f32), e = half a step of a 16-bit type
(f16 2^-11, bf16 2^-8), n keys, D dims, per row and head
  A = max_j scale * sum_d |q_d k_jd|,  B = sum_j p_j |v_j| / sum_j p_j  (per dim)
score: D products summed in f32 in any order err by at most D u A; the parts
  an f32 q is split into leave 2^-22 (f16) or 2^-24 of it, at most 4 u A; the
  factor to log2 units and its product 3 u A.  Scores in [-A, A]: the
  subtraction of the maximum errs by u 2 A and e^x by 2 u more, so each weight's
  relative error is at most  d = ((D + 4 + 3 + 2) A + 4) u, and (1 + d)^2 - 1 with
  its maximum's and the rescaling's alike.  Both sums' n terms add n u each, the
  merge of partial results a few u: 16.
weights as factors of V: parts of an f32 weight leave 2^-22; a 16-bit call's
  decode keeps two parts (f16 2^-22, bf16 2^-16), its prefill one (e).  f16 parts
  have steps of 2^-24 at least: an absolute 2^-25 of a weight whose largest is
  2^15 in a decode, 2^8 or more in a prefill, times the n values of V.
output: rounded to a 16-bit type, e |out| (and e times its smallest normal).
So  |got - want| <= (2 (d + n u) + 16 u + w) B + n f max |v|  (+ e |want|).
"""
import numpy as np

F32, F16, BF16 = 0, 1, 30
U = 2.0 ** -24
HALF = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -126, F16: 2.0 ** -14, BF16: 2.0 ** -126}


def to_bits(x, dt):
    """Round f32 values to dt (nearest even); the storage array."""
    x = np.ascontiguousarray(x, np.float32)
    if dt == F32:
        return x
    if dt == F16:
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r)


def from_bits(a, dt):
    if dt == F32:
        return np.asarray(a, np.float32)
    if dt == F16:
        return a.view(np.float16).astype(np.float32)
    return (a.astype(np.uint32) << 16).view(np.float32)


NAN = {F16: 0x7e00, BF16: 0x7fc0}


class Pool:
    """A page pool of NaN on the host, and scattered pages for sequences of the
    given lengths (page tables padded with ids far outside the pool)."""

    def __init__(self, rng, lens, page_size, n_kv_heads, head_dim, dt, spare=3, width=0):
        need = [-(-max(0, n) // page_size) for n in lens]
        self.ps, self.hk, self.d, self.dt = page_size, n_kv_heads, head_dim, dt
        self.n_pages = sum(need) + spare
        self.k = np.full((self.n_pages, n_kv_heads, page_size, head_dim), NAN[dt], np.uint16)
        self.v = self.k.copy()
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max(width, max(need, default=0), 1)), 1 << 30, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n

    def put(self, s, pos, k, v):
        """Rows k, v [m, hk, d] (f32) at positions pos [m] of sequence s."""
        page, slot = self.table[s, pos // self.ps], pos % self.ps
        self.k[page, :, slot] = to_bits(k, self.dt)
        self.v[page, :, slot] = to_bits(v, self.dt)

    def get(self, s, n):
        page, slot = self.table[s, np.arange(n) // self.ps], np.arange(n) % self.ps
        return from_bits(self.k[page, :, slot], self.dt), from_bits(self.v[page, :, slot], self.dt)

    def fill(self, rng, s, n, std=1.0):
        if n > 0:
            self.put(s, np.arange(n), *(rng.standard_normal((2, n, self.hk, self.d)) * std).astype(np.float32))


def attend(q, k, v, pos, scale):
    """q [m, H, D] over k, v [n, hk, D], row i sees keys 0 .. pos[i]: (out, A, B,
    max |v|) in 64 bits, out zeros where pos < 0."""
    m, H, D = q.shape
    hk, pos = k.shape[1], np.asarray(pos)
    out, A, B = np.zeros((m, H, D)), np.zeros((m, H, 1)), np.zeros((m, H, D))
    q, k, v = (a.astype(np.float64) for a in (q, k, v))
    n = int(pos.max(initial=-1)) + 1
    if n <= 0:
        return out, A, B, 0.0
    seen = np.arange(n)[None] <= pos[:, None]
    some = seen.any(1)
    for h in range(H):
        kk, vv = k[:n, h * hk // H], v[:n, h * hk // H]
        s = np.where(seen, q[:, h] @ kk.T * scale, -np.inf)
        A[:, h, 0] = np.where(seen, np.abs(q[:, h]) @ np.abs(kk).T * abs(scale), 0).max(1)
        p = np.exp(s - np.where(some, s.max(1), 0.0)[:, None])
        p /= np.where(some, p.sum(1), 1.0)[:, None]
        out[:, h], B[:, h] = p @ vv, p @ np.abs(vv)
    return out, A, B, np.abs(v).max(initial=0.0)


def bound(out, A, B, V, n, D, act, cache, prefill):
    d = ((D + 9) * A + 4) * U
    w = 2.0 ** -22 if act == F32 else HALF[act] if prefill else 2.0 ** (-22 if cache == F16 else -16)
    f = 2.0 ** (-33 if prefill else -40) if cache == F16 else 0.0
    tol = (2 * (d + n * U) + 16 * U + w) * B + n * f * V
    return tol + (0 if act == F32 else HALF[act] * (np.abs(out) + tol + TINY[act]))


def rotate(x, c, s):
    """rope_f32 rotate-half in f32: x [m, H, D], c and s [m, D]."""
    half = x.shape[-1] // 2
    c, s = c[:, None], s[:, None]
    lo, hi = x[..., :half], x[..., half:]
    return np.concatenate([lo * c[..., :half] - hi * s[..., :half], hi * c[..., half:] + lo * s[..., half:]], -1)


def tables(n, d, base=10000.0):
    a = np.arange(n)[:, None] * base ** (-2.0 * np.arange(d // 2) / d)
    return tuple(np.concatenate([f(a)] * 2, 1).astype(np.float32) for f in (np.cos, np.sin))
