"""Refusals of the paged KV cache entry points at the ends of their ranges, and the
bounds that their grids and workspaces are sized by."""
import ctypes as C

import pytest

import fuel_amd as F
from fuel_amd._native import lib
from test_paged_cpu import INVALID, UNSUPPORTED, WORKSPACE, append, attend, batch, kv, passes


def test_append_in_place_keeps_its_rows_apart():
    for b in (batch(), batch(rows=3, row_start=None)):
        assert append(b=b, ldq=520, ldqo=512) == INVALID and b"in place" in lib().frq_last_error()
        assert append(b=b, ldq=512, ldqo=520) == INVALID
        assert passes(append(b=b, ldq=520, ldqo=520))
        assert passes(append(b=b, q=1 << 20, q_out=1 << 21, ldq=520, ldqo=512))
