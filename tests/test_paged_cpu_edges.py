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


def _strides(r, h):
    return (ctypes.c_int64 * 2)(r, h)


# memory of a step's rows, in elements: 5 rows, heads of 128
WIDE = 1024   # q rows of 8 heads
A = 1 << 20   # somewhere


@pytest.mark.parametrize("q,q_out,refused", [
    (A, A, False),                             # in place
    (A, A + 2 * 5 * WIDE, False),              # right behind q
    (A, A + 2 * (5 * WIDE - 1), True),         # one element shared
    (A, A + 2 * WIDE, True),                   # a row further
    (A + 2 * 128, A, True),                    # a head before
    (A + 2 * 5 * WIDE, A, False),
])
def test_outputs_that_overlap_queries(q, q_out, refused):
    qs = _strides(WIDE, 128)
    rc = append(paged(), batch(), q=q, q_heads=8, qs=qs, q_out=q_out)
    assert (rc == _lib.ERR_ARG and "overlaps" in error()) == refused
    fn = _lib.lib().kvq_paged_sdpa_prefill
    rc = fn(ctypes.byref(paged()), ctypes.byref(batch()), q, 8, qs, 1.0, 0, 0, q_out, None, 0, None)
    assert (rc == _lib.ERR_ARG and "overlaps" in error()) == refused


def test_outputs_that_overlap_keys_and_values():
    L = _lib.lib()

    def call(k, v, ks, q_out, rows=5):
        return L.kvq_paged_append(ctypes.byref(paged()), ctypes.byref(batch(rows=rows)), k, v, ks, ks, None,
                                  1 << 30, 8, _strides(WIDE, 128), q_out, None)

    def refused(rc):
        return rc == _lib.ERR_ARG and "overlaps" in error()

    ks = _strides(256, 128)
    far = 1 << 28
    for other in (A, A + 2 * (5 * 256 - 1), A - 2 * (5 * WIDE - 1)):
        assert refused(call(A, far, ks, other)) and refused(call(far, A, ks, other))
    for other in (A + 2 * 5 * 256, A - 2 * 5 * WIDE):
        assert not refused(call(A, far, ks, other)) and not refused(call(far, A, ks, other))
    # rows far apart: q_out lies between two of them, or meets the second head of the third
    ks = _strides(100000, 128)
    assert not refused(call(A, far, ks, A + 2 * 256))
    assert not refused(call(A, far, ks, A + 2 * (200000 + 256)))
    assert refused(call(A, far, ks, A + 2 * (200000 + 255)))
    assert refused(call(A, far, ks, A + 2 * (200000 - 5 * WIDE + 1)))
    assert not refused(call(A, far, ks, A + 2 * (200000 - 5 * WIDE)))
    # rows that go backwards, and one row for all
    back = _strides(-100000, 128)
    assert refused(call(A + 2 * 400000, far, back, A + 2 * 200000))
    assert not refused(call(A + 2 * 400000, far, back, A + 2 * 256))
    same = _strides(0, 128)
    assert refused(call(A, far, same, A + 2 * 255)) and not refused(call(A, far, same, A + 2 * 256))
    # a fused projection's rows in place: one row
    assert not refused(call(A + 2 * WIDE, A + 2 * (WIDE + 256), _strides(WIDE + 512, 128), A, rows=1))


def test_queries_that_are_not_contiguous_are_not_rotated_or_answered_in_place():
    fn = _lib.lib().kvq_paged_sdpa_prefill
    for qs in (_strides(WIDE + 8, 128), _strides(WIDE, 64), _strides(0, 128)):
        rc = fn(ctypes.byref(paged()), ctypes.byref(batch()), A, 8, qs, 1.0, 0, 0, A, None, 0, None)
        assert rc == _lib.ERR_ARG and "overlaps" in error()


def test_remembered_workspace_sizes_are_bounded():
    """A server whose steps bring ever new counts of rows."""
    import torch

    import kvq
    cache = object.__new__(kvq.PagedQuantizedKVCache)
    cache._index, cache.device, cache.dtype, cache.head_dim = -1, torch.device("cpu"), torch.float16, 64
    cache._ref, cache._ws_bytes = None, {}
    asked = []
    cache._stream = lambda stream: 0
    cache._workspace = lambda batch, heads, decode: asked.append(batch.rows) or 16
    lens, cu = torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    buf = torch.zeros(9000, 1, 64, dtype=torch.float16)
    call = lambda n: cache._sdpa(lambda *a: 0, buf[:n], table, lens, cu, 1.0, 0, 0, buf[:n], None, None)
    for n in range(9000):
        call(n)
        call(n)  # known by now
    assert asked == list(range(9000))
    assert len(cache._ws_bytes) <= 4096
