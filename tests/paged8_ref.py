"""The 8-bit paged KV cache on the host: e4m3 codes and e8m0 scales as the entry
points define them, and the bounds its attention is held to.

Values.  code * 2^(b - 127): exact in 64 bits, and in the 32 that appended rows have.

Bounds: paged_ref.py's, with these terms in the place of its.
score: a code is exact as an f16 or bf16 operand and a scale is a power of two, so
  the products err as those of a 16-bit cache do; one factor more, exactly.
weights as factors of V: in tiles of 16 rows (decode) bf16 parts, half a step 2^-8 each:
  of f32 rows three (2^-24; 2^-22 is allowed), of others two (2^-16).  In tiles of 128
  rows as a 16-bit cache's: f32 rows two of f16 (2^-22), others one of their own type;
  f16 parts have steps of 2^-24, 2^-25 of a weight whose largest is 2^8 or more, times
  the n values of V.
"""
import numpy as np

import paged_ref as R
from paged_ref import F32, HALF, TINY, U

_c = np.arange(256)
_e, _m = (_c >> 3) & 15, _c & 7
CODE = np.where(_e > 0, (8.0 + _m) * 2.0 ** (_e - 10.0), _m * 2.0 ** -9) * np.where(_c < 128, 1, -1)
CODE[[0x7f, 0xff]] = np.nan
NAN = 0x7f


def scale(b):
    return np.where(b == 255, np.nan, 2.0 ** (np.asarray(b, np.float64) - 127))


def byte(amax):
    """The least byte under which amax is at most 448."""
    amax = np.asarray(amax, np.float64)
    b = np.clip(np.floor(np.log2(np.maximum(amax, 1e-60) / 448)) + 126, 0, 254).astype(np.int64)  # (no more than it)
    while (amax > 448 * scale(b)).any():
        b = b + (amax > 448 * scale(b))
    return b


def encode(x, b):
    """The nearest codes of x under byte b (broadcast), ties to even; infinite and NaN
    values: NaN.  Under the last byte no code stands for a number past f32's."""
    x, s = np.asarray(x, np.float64), scale(b)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = x / s
        y = np.where((np.asarray(b) >= 247) & np.isfinite(y), np.clip(y, -240, 240), y)
        a = np.abs(y)
        step = 2.0 ** np.maximum(np.floor(np.log2(np.where(a > 0, a, 1))) - 3, -9)
        a = np.round(a / step) * step  # (np.round: ties to even; a step of the power of two below)
    pos = CODE[:127]
    code = np.searchsorted(pos, np.where(np.isfinite(a), a, 0))
    code = np.minimum(code, 126)
    assert (np.where(np.isfinite(a), pos[code] - a, 0) == 0).all()
    return np.where(np.isfinite(y), code + np.where(np.signbit(x), 128, 0), NAN).astype(np.uint8)


def same(a, b):
    """Codes that are alike: NaN is one number of two codes."""
    return (a == b) | (((a & 0x7f) == NAN) & ((b & 0x7f) == NAN))


class Pool:
    """A pool of NaN codes and NaN scales on the host, and scattered pages for
    sequences of the given lengths."""

    def __init__(self, rng, lens, page_size, n_kv_heads, head_dim, spare=3, width=0):
        need = [-(-max(0, n) // page_size) for n in lens]
        self.ps, self.hk, self.d = page_size, n_kv_heads, head_dim
        self.n_pages = sum(need) + spare
        self.code = np.full((2, self.n_pages, n_kv_heads, page_size, head_dim), NAN, np.uint8)
        self.scale = np.full((2, self.n_pages, n_kv_heads, page_size // 16), 255, np.uint8)
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max(width, max(need, default=0), 1)), 1 << 30, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n

    def append(self, s, pos0, k, v):
        """Rows k, v [m, hk, d] (f32) at positions pos0 .. of sequence s."""
        end = pos0 + len(k)
        if pos0 % 16 == 0 and end - pos0 >= 64:  # all full blocks at once
            n = (end - pos0) // 16
            j = pos0 + 16 * np.arange(n)
            page, i = self.table[s, j // self.ps], j % self.ps
            ok = (page >= 0) & (page < self.n_pages)
            for w, x in enumerate((k, v)):
                x = np.asarray(x[:16 * n], np.float32).reshape(n, 16, self.hk, self.d).transpose(0, 2, 1, 3)[ok]
                a = np.abs(x)
                b = byte(np.where(np.isfinite(a), a, 0).max((2, 3)))
                code = encode(x, b[..., None, None])
                for t, (pg, at) in enumerate(zip(page[ok], i[ok])):
                    self.code[w, pg, :, at:at + 16] = code[t]
                    self.scale[w, pg, :, at // 16] = b[t]
            pos0, k, v = pos0 + 16 * n, k[16 * n:], v[16 * n:]
        for j0 in range(pos0 // 16 * 16, end, 16):
            lo, hi = max(j0, pos0), min(j0 + 16, end)
            page, i = self.table[s, j0 // self.ps], j0 % self.ps
            if not 0 <= page < self.n_pages:
                continue
            for w, x in enumerate((k, v)):
                x = np.asarray(x[lo - pos0:hi - pos0], np.float32).transpose(1, 0, 2)  # [hk, rows, d]
                a = np.abs(x)
                b = byte(np.where(np.isfinite(a), a, 0).max((1, 2)))
                code = self.code[w, page, :, i:i + 16]
                if lo > j0:
                    was = self.scale[w, page, :, i // 16].astype(np.int64)
                    b = np.where(was == 255, b, np.maximum(b, was))
                    old = CODE[code[:, :lo - j0]] * (scale(was) / scale(b))[:, None, None]
                    code[:, :lo - j0] = encode(old, 127)
                code[:, lo - j0:hi - j0] = encode(x, b[:, None, None])
                self.scale[w, page, :, i // 16] = b

    def get(self, s, n):
        page, at = self.table[s, np.arange(n) // self.ps], np.arange(n) % self.ps
        return tuple(CODE[self.code[w, page, :, at]] * scale(self.scale[w, page, :, at // 16])[..., None]
                     for w in range(2))

    def fill(self, rng, s, n, std=1.0):
        if n > 0:
            self.append(s, 0, *(rng.standard_normal((2, n, self.hk, self.d)) * std).astype(np.float32))


def bound(out, A, B, V, n, D, act, tiles):
    """V: the largest |v| of the n keys."""
    d = ((D + 10) * A + 4) * U
    w = 2.0 ** -22 if act == F32 else HALF[act] if tiles else 2.0 ** -16
    tol = (2 * (d + n * U) + 16 * U + w) * B + TINY[R.BF16]
    if tiles and act != R.BF16:
        tol = tol + n * 2.0 ** -33 * V
    return tol + (0 if act == F32 else HALF[act] * (np.abs(out) + tol + TINY[act]))
