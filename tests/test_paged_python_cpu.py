"""What the Python mirror of the paged KV cache refuses before a call."""
import numpy as np
import pytest

import fuel_amd as F
from fuel_amd.backend import RocmStorage

P = 1 << 20  # an address that nothing reads


class Dev:
    """A device that no call reaches."""

    def __init__(self, ordinal=0):
        self.ordinal = ordinal

    @property
    def handle(self):
        return None


def storage(nbytes, dtype=np.uint16, dev=None):
    """A storage of that many bytes, without device memory."""
    s = object.__new__(RocmStorage)
    s.dev, s.dtype, s.nbytes, s.ptr = dev or DEV, np.dtype(dtype), nbytes, P
    s.shape = (nbytes // s.dtype.itemsize,)
    s.free = lambda: None
    return s


DEV = Dev()


def refused(f, *a, **k):
    with pytest.raises(F.FuelRocmError) as e:
        f(*a, **k)
    assert e.value.status != 0
    return str(e.value)


@pytest.mark.parametrize("x", [np.array([P]), np.array(P), 1.5, "1048576", True, [P], np.zeros(4, np.float32)])
def test_operands_that_are_no_addresses(x):
    """Arrays and tensors of one element have an int() of their value."""
    refused(F.PagedKvCache, DEV, 9, 16, 2, 128, F.F16, x, P)
    for name in ("page_table", "kv_len", "row_start"):
        refused(F.PagedBatch, **dict(dict(page_table=P, kv_len=P, n_seqs=3, max_pages=4, row_start=P), **{name: x}))
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, P, P), F.PagedBatch(P, P, 3, 4)
    for name in ("q", "k", "v", "q_out", "rope_cos", "rope_sin"):
        a = dict(q=P, k=P, v=P, q_out=P, rope_cos=P, rope_sin=P)
        a[name] = x
        refused(F.paged_append, cache, one, F.F16, 4, rope_rows=4, **a)
    for fn in (F.paged_attention_decode, F.paged_attention_prefill):
        refused(fn, cache, one, F.F16, 4, x, P, 0.1)
        refused(fn, cache, one, F.F16, 4, P, x, 0.1)


def test_addresses_reach_the_library():
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, np.int64(P), P), F.PagedBatch(P, np.uint64(P), 3, 4)
    assert cache.struct.k == P and one.struct.kv_len == P and one.struct.row_start is None
    assert "null device handle" in refused(F.paged_append, cache, one, F.F16, 4, P, P, P, P)


def test_workspace_is_a_storage_or_an_address_of_so_many_bytes():
    cache, one = F.PagedKvCache(DEV, 9, 16, 2, 128, F.F16, P, P), F.PagedBatch(P, P, 3, 1 << 16)
    need = F.paged_attention_workspace(cache, one, 4)
    assert need > 0
    for fn in (F.paged_attention_decode, F.paged_attention_prefill):
        args = (cache, one, F.F16, 4, P, P, 0.1)
        for work in (None, P, storage(need - 1, np.uint8)):
            assert "workspace" in refused(fn, *args, work)
        assert "workspace" in refused(fn, *args, P, work_bytes=need - 1)
        refused(fn, *args, np.zeros(need, np.uint8), work_bytes=need)
        assert "null device handle" in refused(fn, *args, P, work_bytes=need)
        assert "null device handle" in refused(fn, *args, storage(need, np.uint8))
