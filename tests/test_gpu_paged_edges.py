"""Calls of the paged cache at the edges of what its documentation allows, on
the GPU against the plain 64-bit implementation of tests/paged_ref.py."""
import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _kvq():
    import kvq
    return kvq


def _cache(ref):
    kvq = _kvq()
    return kvq.PagedQuantizedKVCache(ref.pool.shape[0], ref.page, ref.heads, ref.d, ref.gs,
                                     ref.bits, ref.dt, pool=ref.pool.cuda())


def _cu(rows):
    return [0] + list(np.cumsum(rows))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pages(lens, page):
    return sum(-(-max(n, 0) // page) for n in lens) + 3


# --------------------------------------------------------- where out begins --

OUT = [
    # dt, bits, gs, Hq, Hkv, D, page, lens, rows (None: decode)
    (F16, 4, 64, 8, 2, 128, 16, [1000, 1, 17], None),     # 4 columns a block
    (BF16, 8, 64, 16, 2, 64, 32, [700, 0, 90], None),     # 8
    (F16, 8, 32, 16, 1, 128, 16, [300], None),            # 16
    (F16, 4, 64, 8, 2, 128, 16, [100, 40], [6, 3]),       # drafts
    (BF16, 4, 64, 8, 2, 128, 16, [700, 300], [257, 300]),
    (F16, 8, 64, 4, 2, 256, 32, [400, 130], [130, 100]),
    (BF16, 8, 64, 16, 8, 256, 32, [2000, 1500], [600, 500]),  # units held whole and cut
]


@pytest.mark.parametrize("case", OUT, ids=lambda c: "-".join(str(x) for x in c[1:]))
@pytest.mark.parametrize("cut", [1, 2, 3, 4])
def test_out_may_start_at_any_element(case, cut):
    """The same bits wherever a contiguous `out` starts in its buffer, and
    nothing written beside it."""
    dt, bits, gs, hq, hkv, d, page, lens, rows = case
    gen = torch.Generator().manual_seed(31)
    ref = R.random_pool(gen, _pages(lens, page), page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, ref.pool.shape[0]).cuda()
    cache = _cache(ref)
    n = len(lens) if rows is None else sum(rows)
    q = torch.randn(n, hq, d, generator=gen).to(dt).cuda()

    def call(out):
        if rows is None:
            return cache.sdpa_decode(q, table, _i32(lens), 0.1, out=out)
        return cache.sdpa_prefill(q, table, _i32(lens), _i32(_cu(rows)), 0.1, out=out)

    want = call(torch.zeros(n, hq, d, dtype=dt, device="cuda"))
    buf = torch.full((n * hq * d + 8,), 7.0, dtype=dt, device="cuda")
    out = buf[cut:cut + n * hq * d].view(n, hq, d)
    assert out.data_ptr() % 16 == 2 * cut
    assert call(out) is out
    cache.check()
    assert torch.equal(out.view(torch.int16), want.view(torch.int16))
    assert (buf[:cut] == 7.0).all() and (buf[cut + n * hq * d:] == 7.0).all()


@pytest.mark.parametrize("case", OUT, ids=lambda c: "-".join(str(x) for x in c[1:]))
def test_out_may_be_q(case):
    dt, bits, gs, hq, hkv, d, page, lens, rows = case
    gen = torch.Generator().manual_seed(33)
    ref = R.random_pool(gen, _pages(lens, page), page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, ref.pool.shape[0]).cuda()
    cache = _cache(ref)
    n = len(lens) if rows is None else sum(rows)
    q = torch.randn(n, hq, d, generator=gen).to(dt).cuda()

    def call(q, out=None):
        if rows is None:
            return cache.sdpa_decode(q, table, _i32(lens), 0.1, out=out)
        return cache.sdpa_prefill(q, table, _i32(lens), _i32(_cu(rows)), 0.1, out=out)

    want = call(q)
    for _ in range(5):
        x = q.clone()
        assert torch.equal(call(x, x).view(torch.int16), want.view(torch.int16))
    with pytest.raises(_kvq().KvqError, match="overlaps"):
        buf = torch.zeros((n + 1) * hq * d, dtype=dt, device="cuda")
        call(buf[:n * hq * d].view(n, hq, d), buf[hq:hq + n * hq * d].view(n, hq, d))


# ------------------------------------------------------- streams and the flag --

def _small(seed=32, n=40):
    gen = torch.Generator().manual_seed(seed)
    ref = R.random_pool(gen, 6, 16, 2, 64, 64, 4, F16)
    table = R.make_table(gen, [n], 16, 6)
    return gen, ref, table, _cache(ref)


def test_check_takes_what_is_raised_by_then():
    """Errors are reported once, by the first check after them; one that another
    stream raises later is the next check's."""
    kvq = _kvq()
    gen, ref, table, cache = _small()
    k = torch.randn(1, 2, 64, generator=gen).to(F16).cuda()
    good, bad = _i32([40]), _i32([4000])  # a position past the table
    dtab = table.cuda()
    cache.append(k, k, dtab, bad)
    with pytest.raises(kvq.KvqError):
        cache.check()
    cache.check()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s2):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        cache.append(k, k, dtab, bad)
    with torch.cuda.stream(s1):
        cache.append(k, k, dtab, good)
        cache.check()               # nothing of s1's; s2 has not come to its append
    with torch.cuda.stream(s2):
        with pytest.raises(kvq.KvqError):
            cache.check()
    with torch.cuda.stream(s1):
        cache.check()
    cache._status.fill_(3)          # both kinds at once: the wait that ran out is told
    with pytest.raises(kvq.KvqError, match="waiting"):
        cache.check()
    cache.check()


CAPTURE = """
import torch, sys
sys.path[:0] = [%r, %r]
import kvq, paged_ref as R
import test_gpu_paged_edges as T
gen, ref, table, cache = T._small()
q = torch.randn(3, 8, 64, generator=gen).to(torch.float16).cuda()
lens, cu, dtab = T._i32([38]), T._i32([0, 3]), table.cuda()
kw = dict(window=20, sinks=2)
out = [torch.zeros_like(q) for _ in range(2)]
out1 = torch.zeros(1, 8, 64, dtype=torch.float16, device="cuda")
side = torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=side):
    for o in out:  # the library's own workspaces, of a stream that is being captured
        cache.sdpa_prefill(q, dtab, lens, cu, 0.1, out=o, stream=side.cuda_stream, **kw)
    cache.sdpa_decode(q[2:], dtab, lens, 0.1, out=out1, stream=side.cuda_stream, **kw)
for n in (38, 40, 35):
    lens.fill_(n)
    for o in out + [out1]:
        o.zero_()
    g.replay()
    torch.cuda.synchronize()
    cache.check()
    want = cache.sdpa_prefill(q, dtab, lens, cu, 0.1, **kw)
    assert torch.equal(out[0], want) and torch.equal(out[1], want)
    assert torch.equal(out1, cache.sdpa_decode(q[2:], dtab, lens, 0.1, **kw))
print("captured")
"""


def test_capture_with_the_librarys_workspaces():
    """The first call of a process that needs the library's own memory may come
    while its stream is being captured."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = CAPTURE % (here, os.path.join(os.path.dirname(here), "mlx-bun_b200"))
    env = dict(os.environ, PYTHONPATH=os.path.dirname(here))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
