"""More refusals of the paged cache's C entry points, which come before any
CUDA call."""
import ctypes

import pytest

from kvq import _lib
from test_paged_cpu import S2, append, batch, error, paged, sdpa


@pytest.mark.parametrize("what", ["status", "page_table", "seq_lens", "cu_rows"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_of_a_step_are_aligned_to_their_elements(what, off):
    p = paged(**{what: 4096 + off}) if what == "status" else paged()
    b = batch() if what == "status" else batch(**{what: 4096 + off})
    for rc in (append(p, b), sdpa(p, b)):
        assert rc == _lib.ERR_ARG and "aligned" in error()


def test_rows_are_aligned_to_their_elements():
    qs = (ctypes.c_int64 * 2)(1024, 128)
    for kw in (dict(k=4097), dict(v=4097), dict(q=4097, q_heads=8, qs=qs, q_out=8192),
               dict(q=4096, q_heads=8, qs=qs, q_out=8193)):
        assert append(paged(), batch(), **kw) == _lib.ERR_ARG and "aligned" in error()
    for off in (1, 2, 3):
        r = _lib.RopeArgs(64, 0, 1e4, 1.0, 1.0, 4096 + off)
        assert append(paged(), batch(), r) == _lib.ERR_ARG and "aligned" in error()
    for kw in (dict(q=4097), dict(out=4097)):
        for decode in (False, True):
            b = batch(rows=2) if decode else batch()
            assert sdpa(paged(), b, decode=decode, **kw) == _lib.ERR_ARG and "aligned" in error()
