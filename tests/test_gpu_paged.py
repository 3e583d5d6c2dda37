"""The paged cache on the GPU against the plain 64-bit implementation of
tests/paged_ref.py: codes, scales, biases and rotated queries bit for bit,
attention within the tolerance that paged_ref.tolerance derives."""
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


def _check(got, want, mag, magc, l1, dt, dense=False):
    d = (got.double().cpu() - want).abs()
    tol = R.tolerance(want, mag, magc, l1, dt, dense)
    bad = d > tol
    if bool(bad.any()):
        raise AssertionError(f"{int(bad.sum())} outside, up to {float((d / tol).max()):.3f} times")
    assert bool(torch.isfinite(got).all())


# ------------------------------------------------------------------ append --

APPEND = [
    # dt, bits, gs, Hq, Hkv, D, page, lens, rows, pad, rope
    (F16, 8, 64, 16, 4, 128, 64, [2048], [1], 0, dict(dims=128)),
    (BF16, 4, 64, 8, 2, 128, 16, [17, 1, 300, 16], [1, 1, 1, 1], 0, dict(dims=128, base=5e5)),
    (BF16, 8, 64, 4, 2, 256, 32, [70, 131072, 33, 5], [33, 7, 33, 0], 5, dict(dims=128)),
    (F16, 4, 32, 3, 1, 64, 16, [100, 9], [100, 2], 1, dict(dims=64, traditional=True)),
    (F16, 8, 128, 2, 2, 128, 128, [257], [200], 0, dict(dims=20)),
    (BF16, 4, 128, 6, 3, 256, 256, [513, 1], [300, 1], 3, dict(dims=12, traditional=True)),
    (BF16, 8, 32, 8, 8, 64, 64, [65], [64], 0, dict(dims=0)),
    (F16, 4, 64, 5, 5, 64, 32, [40, 20], [13, 20], 0,
     dict(dims=32, scale=0.25, pre=1.2079441, table=True)),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x) for x in c[1:7]))
@pytest.mark.parametrize("layout", ["fused", "odd", "in place"])
def test_append(case, layout):
    dt, bits, gs, hq, hkv, d, page, lens, rows, pad, rope = case
    kvq = _kvq()
    gen = torch.Generator().manual_seed(5)
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, pages)
    cache = _cache(ref)
    cu = _cu(rows)
    T = cu[-1] + pad
    if layout == "odd":  # rows at odd strides: no wide loads
        buf = torch.randn(T, (hq + 2 * hkv) * d + 3, generator=gen).to(dt).cuda()[:, 1:-2]
        buf = buf.unflatten(1, (hq + 2 * hkv, d))
    else:
        buf = torch.randn(T, hq + 2 * hkv, d, generator=gen).to(dt).cuda()
    q, k, v = buf[:, :hq], buf[:, hq:hq + hkv], buf[:, hq + hkv:]
    if layout == "in place":
        q = q.contiguous()
    hq_, hk_, hv_ = q.cpu(), k.cpu(), v.cpu()
    dims = rope["dims"]
    freqs = None
    if rope.get("table"):
        freqs = (10000.0 ** (torch.arange(dims // 2) / (dims / 2))).float()
        freqs[-1] = float("inf")
    kw = dict(base=rope.get("base", 1e4), scale=rope.get("scale", 1.0),
              traditional=rope.get("traditional", False))
    spec = kvq.Rope(dims, freqs=freqs.cuda() if freqs is not None else None,
                    pre_scale=rope.get("pre", 1.0), **kw)
    q_out = q if layout == "in place" else torch.full((T, hq, d), 7.0, dtype=dt, device="cuda")
    got = cache.append(k, v, table.cuda(), _i32(lens), _i32(cu), rope=spec, q=q, q_out=q_out)
    assert got is q_out
    cache.check()
    want_q = hq_.clone() if layout == "in place" else torch.full((T, hq, d), 7.0, dtype=dt)
    for b, n in enumerate(lens):
        r0, r1 = cu[b], cu[b + 1]
        if r1 == r0:
            continue
        pos = torch.arange(n - (r1 - r0), n)
        rk = R.rotate(hk_[r0:r1], pos, dims, freqs=freqs, pre=rope.get("pre", 1.0), **kw)
        want_q[r0:r1] = R.rotate(hq_[r0:r1], pos, dims, freqs=freqs, pre=rope.get("pre", 1.0), **kw)
        ref.put(table[b], pos, rk, hv_[r0:r1])
    assert torch.equal(cache.pool.cpu(), ref.pool)
    assert torch.equal(q_out.cpu().view(torch.int16), want_q.view(torch.int16))


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("gs", [32, 64, 128])
def test_append_quantizes_special_groups(dt, bits, gs):
    """Constant, tiny, huge and tie-rich groups get the rule's codes, as
    kvq.quantize gives them and as the oracle does."""
    gen = torch.Generator().manual_seed(19)
    d, hkv, page = 128, 2, 16
    big = 6e4 if dt == F16 else 3e38
    rows = [torch.zeros(d), torch.full((d,), 0.7), torch.full((d,), -3.0), torch.full((d,), big),
            torch.arange(d) - 64.0, torch.arange(d) / 16.0, (torch.arange(d) - 40.0) * 0.375,
            torch.randn(d, generator=gen) * big / 8, torch.randn(d, generator=gen) * 1e-7,
            torch.randint(-15, 16, (d,), generator=gen) * 0.5, -torch.arange(d).float(),
            torch.randn(d, generator=gen).clamp(-1, 1)]
    x = torch.stack(rows).to(dt)[:, None].expand(-1, hkv, -1).contiguous()
    x[:, 1] = x[:, 1].flip(-1)
    ref = R.random_pool(gen, 2, page, hkv, d, gs, bits, dt)
    cache = _cache(ref)
    table = torch.tensor([[1]], dtype=torch.int32)
    cache.append(x.cuda(), x.cuda(), table.cuda(), _i32([12]), _i32([0, 12]))
    ref.put(table[0], torch.arange(12), x, x)
    # bit for bit, but for the payload of the NaN scales of groups with infinities
    for got, want in zip(cache.keys + cache.values, (ref.kc, ref.kp, ref.vc, ref.vp)):
        got = got.cpu()
        if got.dtype == torch.int32:
            assert torch.equal(got, want)
        else:
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan)
            assert torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan])


def test_append_skips_rows_without_a_place():
    """Negative positions, a position past the table and a page outside the
    pool raise the flag and write nothing; the other rows land."""
    gen = torch.Generator().manual_seed(6)
    ref = R.random_pool(gen, 6, 16, 2, 64, 64, 4, F16)
    cache = _cache(ref)
    table = torch.tensor([[0, 1], [2, 3], [4, 9], [5, -1]], dtype=torch.int32)
    lens, cu = [3, 40, 17, 5], [0, 5, 15, 17, 18]
    k = torch.randn(18, 2, 64, generator=gen).to(F16)
    cache.append(k.cuda(), k.cuda(), table.cuda(), _i32(lens), _i32(cu))
    with pytest.raises(_kvq().KvqError):
        cache.check()
    cache.check()
    ref.put(table[0], torch.arange(0, 3), k[2:5], k[2:5])      # rows 0, 1 at positions -2, -1
    ref.put(table[1], torch.arange(30, 32), k[5:7], k[5:7])    # positions 32.. have no entry
    ref.put(table[2], torch.tensor([15]), k[15:16], k[15:16])  # position 16: page 9 of 6
    ref.put(table[3], torch.tensor([4]), k[17:18], k[17:18])
    assert torch.equal(cache.pool.cpu(), ref.pool)


# ------------------------------------------------------------------ decode --

DECODE = [
    # dt, bits, gs, Hq, Hkv, D, page, lens, window, sinks
    (F16, 8, 64, 16, 4, 128, 64, [2048], 0, 0),
    (F16, 4, 64, 32, 8, 128, 16, [1000, 1, 17, 333], 0, 0),
    (BF16, 4, 64, 32, 8, 128, 64, [1000, 0, 16, 15, 4097], 0, 0),
    (BF16, 8, 64, 8, 4, 256, 32, [1100, 1024, 5, 1025], 1024, 4),
    (F16, 4, 32, 4, 4, 64, 16, [130, 77], 0, 0),
    (F16, 8, 32, 2, 1, 64, 128, [129], 1, 1),
    (BF16, 8, 128, 6, 2, 128, 256, [700, 256], 100, 40),
    (F16, 4, 128, 16, 1, 256, 16, [500, 47, 48], 33, 0),
    (BF16, 4, 64, 24, 1, 64, 32, [222], 0, 0),
    (F16, 8, 64, 20, 1, 128, 16, [95, 3], 17, 20),
    (F16, 4, 64, 5, 1, 128, 64, [9000], 0, 0),
    (BF16, 4, 32, 9, 3, 128, 16, [513] * 7, 64, 3),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(str(x) for x in c))
def test_decode(case):
    dt, bits, gs, hq, hkv, d, page, lens, window, sinks = case
    gen = torch.Generator().manual_seed(7)
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, pages)
    R.poison(ref, table, lens)
    cache = _cache(ref)
    q = torch.randn(len(lens), hq, d, generator=gen).to(dt)
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), d ** -0.5, window, sinks)
    cache.check()
    want = R.attention(ref, q, table, lens, list(range(len(lens) + 1)), d ** -0.5, window, sinks)
    _check(got, *want, dt)
    for b, n in enumerate(lens):
        if n == 0:
            assert not got[b].any()


@pytest.mark.parametrize("kind", ["decode", "drafts", "chunks"])
def test_many_sequences(kind):
    """More sequences and column blocks than a plan in shared memory holds, with
    empty ones among them, through both attention kernels."""
    gen = torch.Generator().manual_seed(20)
    B, page, hq, hkv, d, dt = 600, 16, 8, 2, 64, F16
    lens = torch.randint(0, 40, (B,), generator=gen).tolist()
    lens[7] = lens[599] = 0
    if kind == "decode":
        rows = [1] * B
    else:
        most = 4 if kind == "drafts" else 40
        rows = [int(torch.randint(0, most + 1, (1,), generator=gen)) for _ in range(B)]
        if kind == "chunks":  # past 64 rows * heads of a group on average
            rows = [max(r, 17) for r in rows]
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, 32, 4, dt)
    table = R.make_table(gen, lens, page, pages)
    cache = _cache(ref)
    cu = _cu(rows)
    q = torch.randn(cu[-1], hq, d, generator=gen).to(dt)
    if kind == "decode":
        got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), 0.2)
    else:
        got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), 0.2, 24, 2)
    cache.check()
    window = (0, 0) if kind == "decode" else (24, 2)
    # rows before a sequence's first token see nothing
    want = [torch.zeros(cu[-1], hq, n, dtype=torch.float64) for n in (d, d, d, 1)]
    for b, n in enumerate(lens):
        skip = max(0, rows[b] - n)
        if rows[b] > skip:
            r0, r1 = cu[b] + skip, cu[b + 1]
            for w, x in zip(want, R.attention(ref, q[r0:r1], table[b:b + 1], [n], [0, r1 - r0], 0.2, *window)):
                w[r0:r1] = x
    _check(got, *want, dt, dense=kind == "chunks")


@pytest.mark.parametrize("window", [64, 65, 2 ** 31 - 1])
def test_window_as_long_as_the_table(window):
    gen = torch.Generator().manual_seed(21)
    ref = R.random_pool(gen, 9, 16, 1, 128, 64, 8, BF16)
    table = R.make_table(gen, [64, 50], 16, 9, extra=0)
    cache = _cache(ref)
    q = torch.randn(90, 2, 128, generator=gen).to(BF16)
    # 60 rows for 50 tokens: ten of them stand before the first
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32([64, 50]), _i32([0, 30, 90]), 0.1, window,
                             2 ** 31 - 1)
    want = R.attention(ref, q[:30], table[:1], [64], [0, 30], 0.1)
    _check(got[:30], *want, BF16, dense=True)
    assert not got[30:40].any()
    want = R.attention(ref, q[40:], table[1:], [50], [0, 50], 0.1)
    _check(got[40:], *want, BF16, dense=True)


def test_decode_strided_queries_and_table():
    gen = torch.Generator().manual_seed(8)
    lens, page, hq, hkv, d = [70, 35], 16, 8, 2, 128
    ref = R.random_pool(gen, 12, page, hkv, d, 64, 4, F16)
    table = R.make_table(gen, lens, page, 12)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    cache = _cache(ref)
    for cut in (0, 1):  # aligned rows, and rows that start at an odd element
        buf = torch.randn(2, (hq + 3) * d + 2 * cut, generator=gen).to(F16).cuda()
        q = buf[:, cut:cut + (hq + 3) * d].unflatten(1, (hq + 3, d))[:, 2:2 + hq]
        got = cache.sdpa_decode(q, wide.cuda()[:, :table.shape[1]], _i32(lens), 0.3)
        want = R.attention(ref, q.cpu(), table, lens, [0, 1, 2], 0.3)
        _check(got, *want, F16)


def test_decode_masks_pages_outside_the_pool():
    gen = torch.Generator().manual_seed(9)
    ref = R.random_pool(gen, 5, 16, 1, 64, 32, 8, BF16)
    cache = _cache(ref)
    table = torch.tensor([[0, 77, 1], [2, 3, 4], [0, 1, 2]], dtype=torch.int32)
    lens = [48, 33, 49]  # the last is longer than its table
    q = torch.randn(3, 2, 64, generator=gen).to(BF16)
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), 0.125)
    with pytest.raises(_kvq().KvqError):
        cache.check()
    skip = torch.tensor([[0, 1]], dtype=torch.int32)  # keys of the two good pages
    want = R.attention(ref, q[:1], skip, [32], [0, 1], 0.125)
    _check(got[:1], *want, BF16)
    want = R.attention(ref, q[1:2], table[1:2], [33], [0, 1], 0.125)
    _check(got[1:2], *want, BF16)
    assert not got[2].any()


@pytest.mark.parametrize("big", [1e4, 6e4])
def test_decode_far_apart_logits(big):
    """Logits of thousands on both sides, and queries near fp16's limits."""
    gen = torch.Generator().manual_seed(10)
    lens, d = [300, 31], 128
    ref = R.random_pool(gen, 24, 16, 2, d, 64, 4, F16)
    table = R.make_table(gen, lens, 16, 24)
    cache = _cache(ref)
    q = torch.randn(2, 8, d, generator=gen)
    q = (q / q.abs().max() * big).to(F16)
    q[1, 3] = 0
    q[1, 4] *= 2.0 ** -20
    scale = 0.01
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), scale)
    want = R.attention(ref, q, table, lens, [0, 1, 2], scale)
    _check(got, *want, F16)


def test_decode_wide_exponents_bf16():
    """bf16 queries, scales and biases far outside fp16's range."""
    gen = torch.Generator().manual_seed(11)
    lens, d = [200, 64], 128
    ref = R.random_pool(gen, 20, 16, 2, d, 64, 8, BF16)
    ref.kp *= 2.0 ** 40
    ref.vp *= 2.0 ** -60
    table = R.make_table(gen, lens, 16, 20)
    cache = _cache(ref)
    q = (torch.randn(2, 4, d, generator=gen) * 2.0 ** -38).to(BF16)
    q[0, 1] = 0
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), 0.1)
    _check(got, *R.attention(ref, q, table, lens, [0, 1, 2], 0.1), BF16)


# ----------------------------------------------------------------- prefill --

PREFILL = [
    # dt, bits, gs, Hq, Hkv, D, page, lens, rows, pad, window, sinks
    (F16, 8, 64, 8, 2, 128, 64, [600], [200], 0, 0, 0),
    (F16, 4, 64, 32, 8, 128, 16, [100, 40, 333, 8], [1, 8, 3, 8], 3, 0, 0),
    (BF16, 4, 64, 8, 2, 128, 16, [700, 1, 300, 64], [257, 1, 300, 0], 9, 100, 4),
    (BF16, 8, 64, 4, 2, 256, 32, [400, 130], [130, 100], 0, 128, 0),
    (F16, 4, 32, 3, 1, 64, 16, [75, 20], [75, 2], 1, 0, 0),
    (F16, 8, 128, 4, 4, 128, 128, [129], [128], 0, 1, 2),
    (BF16, 4, 128, 5, 1, 256, 256, [77], [77], 2, 30, 10),
    (BF16, 8, 32, 16, 1, 128, 16, [250, 250], [3, 90], 0, 0, 0),
    (F16, 8, 32, 24, 1, 64, 64, [150], [40], 0, 16, 1),
    (F16, 4, 64, 8, 2, 128, 64, [3000, 2100], [520, 1030], 0, 0, 0),
    (BF16, 8, 128, 2, 2, 128, 32, [1300], [1300], 4, 256, 300),
    # runs of several tiles in several units per CTA, one and two row tiles
    (BF16, 8, 64, 16, 8, 256, 32, [2000, 1500], [600, 500], 0, 0, 0),
    (F16, 4, 64, 16, 8, 256, 16, [1900, 700], [700, 300], 2, 512, 20),
    (F16, 8, 64, 16, 4, 128, 64, [2100, 1500], [700, 600], 0, 0, 0),
]


@pytest.mark.parametrize("case", PREFILL, ids=lambda c: "-".join(str(x) for x in c))
def test_prefill(case):
    dt, bits, gs, hq, hkv, d, page, lens, rows, pad, window, sinks = case
    gen = torch.Generator().manual_seed(12)
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, pages)
    R.poison(ref, table, lens)
    cache = _cache(ref)
    cu = _cu(rows)
    T = cu[-1] + pad
    q = torch.randn(T, hq, d, generator=gen).to(dt)
    out = torch.full((T, hq, d), 7.0, dtype=dt, device="cuda")
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), d ** -0.5, window,
                             sinks, out=out)
    cache.check()
    assert got is out
    assert (got[cu[-1]:] == 7.0).all()
    want = R.attention(ref, q, table, lens, cu, d ** -0.5, window, sinks)
    _check(got[:cu[-1]], *[x[:cu[-1]] for x in want], dt, dense=True)


def test_prefill_rows_before_the_first_token_see_nothing():
    gen = torch.Generator().manual_seed(13)
    ref = R.random_pool(gen, 8, 16, 2, 128, 64, 8, F16)
    lens, cu = [3, 0, 20], [0, 8, 12, 20]
    table = R.make_table(gen, lens, 16, 8)
    cache = _cache(ref)
    q = torch.randn(20, 4, 128, generator=gen).to(F16)
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), 0.09)
    assert not got[:5].any() and not got[8:12].any()
    for r0, r1, b, n in ((5, 8, 0, 3), (12, 20, 2, 20)):
        want = R.attention(ref, q[r0:r1], table[b:b + 1], [n], [0, r1 - r0], 0.09)
        _check(got[r0:r1], *want, F16, dense=True)


# -------------------------------------------------------------- as a whole --



@pytest.mark.parametrize("dt,bits,window,sinks", [(F16, 4, 0, 0), (BF16, 8, 48, 4)])
def test_append_prefill_decode_with_a_shared_prefix_in_a_graph(dt, bits, window, sinks):
    """Two sequences share their first pages; a ragged prompt chunk, then
    decode steps from one captured graph whose lengths advance on the GPU."""
    kvq = _kvq()
    gen = torch.Generator().manual_seed(14)
    hq, hkv, d, page, gs = 8, 2, 128, 16, 64
    ref = R.random_pool(gen, 32, page, hkv, d, gs, bits, dt)
    cache = _cache(ref)
    rope = kvq.Rope(d, base=1e4)
    table = torch.full((3, 8), -1, dtype=torch.int32)
    table[0] = torch.arange(0, 8)
    table[1, :2] = table[0, :2]          # 32 shared tokens
    table[1, 2:] = torch.arange(8, 14)
    table[2] = torch.arange(20, 28)
    lens, rows = [50, 37, 19], [50, 5, 19]
    cu = _cu(rows)
    scale = d ** -0.5

    def reference_step(lens, rows, q, k, v):
        cu = _cu(rows)
        rq = q.clone()
        for b, n in enumerate(lens):
            pos = torch.arange(n - rows[b], n)
            rq[cu[b]:cu[b + 1]] = R.rotate(q[cu[b]:cu[b + 1]], pos, d)
            ref.put(table[b], pos, R.rotate(k[cu[b]:cu[b + 1]], pos, d), v[cu[b]:cu[b + 1]])
        return rq, R.attention(ref, rq, table, lens, cu, scale, window, sinks)

    # the shared prefix first, then the sequences' own rows
    q, k, v = (torch.randn(cu[-1], h, d, generator=gen).to(dt) for h in (hq, hkv, hkv))
    dtab, dlens, dcu = table.cuda(), _i32(lens), _i32(cu)
    rq = cache.append(k.cuda(), v.cuda(), dtab, dlens, dcu, rope=rope, q=q.cuda())
    got = cache.sdpa_prefill(rq, dtab, dlens, dcu, scale, window, sinks)
    want_q, want = reference_step(lens, rows, q, k, v)
    assert torch.equal(rq.cpu(), want_q)
    assert torch.equal(cache.pool.cpu(), ref.pool)
    _check(got, *want, dt, dense=True)

    sq, sk, sv = (torch.zeros(3, h, d, dtype=dt, device="cuda") for h in (hq, hkv, hkv))
    rq, out = torch.empty_like(sq), torch.empty_like(sq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        dlens.add_(1)
        cache.append(sk, sv, dtab, dlens, rope=rope, q=sq, q_out=rq)
        cache.sdpa_decode(rq, dtab, dlens, scale, window, sinks, out=out)
    for step in range(14):  # crosses page borders
        q, k, v = (torch.randn(3, h, d, generator=gen).to(dt) for h in (hq, hkv, hkv))
        sq.copy_(q), sk.copy_(k), sv.copy_(v)
        g.replay()
        lens = [n + 1 for n in lens]
        want_q, want = reference_step(lens, [1, 1, 1], q, k, v)
        assert torch.equal(rq.cpu(), want_q)
        _check(out, *want, dt)
    assert torch.equal(cache.pool.cpu(), ref.pool)
    cache.check()


def test_decode_equals_prefill_of_one_row():
    gen = torch.Generator().manual_seed(15)
    lens, d = [90, 500, 3], 128
    ref = R.random_pool(gen, 48, 16, 2, d, 64, 4, F16)
    table = R.make_table(gen, lens, 16, 48)
    cache = _cache(ref)
    q = torch.randn(3, 8, d, generator=gen).to(F16).cuda()
    a = cache.sdpa_decode(q, table.cuda(), _i32(lens), 0.1, 64, 4)
    b = cache.sdpa_prefill(q, table.cuda(), _i32(lens), _i32([0, 1, 2, 3]), 0.1, 64, 4)
    want = R.attention(ref, q.cpu(), table, lens, [0, 1, 2, 3], 0.1, 64, 4)
    _check(a, *want, F16)
    _check(b, *want, F16, dense=True)


def test_two_streams_at_once_and_repeat_bitwise():
    """Calls on two streams with the calls' own workspaces, many times over:
    every result equals the first, bit for bit."""
    gen = torch.Generator().manual_seed(16)
    lens, d, page = [4000, 2500, 700], 128, 16
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, 2, d, 64, 4, F16)
    table = R.make_table(gen, lens, page, pages).cuda()
    cache = _cache(ref)
    q1 = torch.randn(3, 8, d, generator=gen).to(F16).cuda()
    q2 = torch.randn(200, 8, d, generator=gen).to(F16).cuda()
    dl, cu = _i32(lens), _i32([0, 90, 91, 200])
    one = cache.sdpa_decode(q1, table, dl, 0.1)
    two = cache.sdpa_prefill(q2, table, dl, cu, 0.1)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    a, b = [], []
    for _ in range(20):
        with torch.cuda.stream(s1):
            a.append(cache.sdpa_decode(q1, table, dl, 0.1))
        with torch.cuda.stream(s2):
            b.append(cache.sdpa_prefill(q2, table, dl, cu, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, one) for x in a)
    assert all(torch.equal(x, two) for x in b)


def test_caller_workspace():
    kvq = _kvq()
    gen = torch.Generator().manual_seed(17)
    lens, d = [900, 40], 128
    ref = R.random_pool(gen, 80, 16, 2, d, 64, 8, F16)
    table = R.make_table(gen, lens, 16, 80).cuda()
    cache = _cache(ref)
    q = torch.randn(2, 8, d, generator=gen).to(F16).cuda()
    dl = _i32(lens)
    n = cache.workspace_bytes(2, 8, table, dl)
    ws = torch.full((n + 64,), 0x5a, dtype=torch.uint8, device="cuda")
    got = cache.sdpa_decode(q, table, dl, 0.1, workspace=ws[:n])
    assert (ws[n:] == 0x5a).all()
    assert torch.equal(got, cache.sdpa_decode(q, table, dl, 0.1))
    if n:
        with pytest.raises(kvq.KvqError):
            cache.sdpa_decode(q, table, dl, 0.1, workspace=ws[:n - 1])


def test_offsets_past_32_bits():
    """Pages that lie more than 2^32 bytes into the pool."""
    kvq = _kvq()
    dt, hq, hkv, d, page, gs, bits = F16, 8, 2, 128, 64, 64, 4
    shape = kvq.PagedQuantizedKVCache.pool_shape(1, page, hkv, d, gs, bits, dt)
    pages = (6 << 30) // (int(np.prod(shape)) * 4)
    pool = torch.empty((pages,) + shape[1:], dtype=torch.int32, device="cuda")
    cache = kvq.PagedQuantizedKVCache(pages, page, hkv, d, gs, bits, dt, pool=pool)
    gen = torch.Generator().manual_seed(18)
    lens = [200, 130]
    small = R.random_pool(gen, 8, page, hkv, d, gs, bits, dt)
    low = torch.arange(8, dtype=torch.int32).view(2, 4)
    high = low + (pages - 8)
    k, v = (torch.randn(330, hkv, d, generator=gen).to(dt) for _ in range(2))
    q = torch.randn(330, hq, d, generator=gen).to(dt)
    cu = [0, 200, 330]
    cache.append(k.cuda(), v.cuda(), high.cuda(), _i32(lens), _i32(cu))
    for b, n in enumerate(lens):
        small.put(low[b], torch.arange(n), k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]])
    for b, n in enumerate(lens):
        pg, tile, row = small.index(low[b], torch.arange(n))
        codes, pairs = cache.keys
        assert torch.equal(codes[(pg + pages - 8).cuda(), :, tile.cuda(), row.cuda()].cpu(),
                           small.kc[pg, :, tile, row])
    got = cache.sdpa_prefill(q.cuda(), high.cuda(), _i32(lens), _i32(cu), 0.09)
    _check(got, *R.attention(small, q, low, lens, cu, 0.09), dt, dense=True)
    q1 = q[[199, 329]]
    got = cache.sdpa_decode(q1.cuda(), high.cuda(), _i32(lens), 0.09)
    _check(got, *R.attention(small, q1, low, lens, [0, 1, 2], 0.09), dt)


def test_nothing_to_do():
    kvq = _kvq()
    cache = kvq.PagedQuantizedKVCache(2, 16, 2, 64, 32, 4, F16)
    t, z = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), _i32([])
    e = torch.empty(0, 2, 64, dtype=F16, device="cuda")
    cache.append(e, e, t, z, q=e)
    assert cache.sdpa_decode(e, t, z, 1.0).shape == (0, 2, 64)
    assert cache.sdpa_prefill(e, t, z, _i32([0]), 1.0).shape == (0, 2, 64)
    cache.check()
