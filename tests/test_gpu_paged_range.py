"""Attention over pages whose scales lie far apart, or are not finite where a
query does not look, on the GPU against the plain 64-bit implementation."""
import pytest
import torch

import paged_chunk_ref as C
import paged_ref as R
from test_gpu_paged import _cache, _check, _cu, _i32, _pages

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _pool(seed, lens, page, hkv, d, gs, bits, dt):
    gen = torch.Generator().manual_seed(seed)
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    return gen, ref, R.make_table(gen, lens, page, pages)


def _row(ref, table, b, pos):
    """Index of position `pos` of sequence b in the pool's parts (all heads)."""
    pg, tile, row = ref.index(table[b], torch.tensor([pos]))
    return int(pg), slice(None), int(tile), int(row)


def _check_after_first(got, ref, q, table, lens, cu, scale, dt, window=0, sinks=0):
    """_check, for rows of which the first of a sequence may see nothing."""
    for b, n in enumerate(lens):
        skip = max(0, cu[b + 1] - cu[b] - n)
        r0, r1 = cu[b] + skip, cu[b + 1]
        assert not got[cu[b]:r0].any()
        want = R.attention(ref, q[r0:r1], table[b:b + 1], [n], [0, r1 - r0], scale, window, sinks)
        _check(got[r0:r1], *want, dt)


# ------------------------------------------------------- few rows a sequence --

FORMS = [
    # Hq, Hkv, D, gs, rows of each sequence (None: single tokens)
    (8, 2, 128, 64, None), (16, 2, 128, 64, None), (16, 1, 128, 32, None), (8, 2, 64, 32, None),
    (4, 2, 256, 64, None), (16, 2, 256, 128, None), (8, 2, 128, 32, [3, 2, 4, 1]),
]


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(x) for x in f[:4]) + ("" if f[4] is None else "-rows"))
@pytest.mark.parametrize("apart", ["zero", 10, 14, 18, 40])
def test_groups_of_v_far_apart(dt, bits, form, apart):
    """One group of every V row far below the others (or all zeros, as the
    append leaves it) keeps its own precision."""
    if apart == 40 and dt == F16:
        pytest.skip("fp16 has no such scale")
    hq, hkv, d, gs, rows = form
    lens = [2048, 700, 33, 1]
    gen, ref, table = _pool(41, lens, 16, hkv, d, gs, bits, dt)
    low = d // gs - 1
    if apart == "zero":
        ref.vp[..., 0] *= 64.0
        ref.vp[..., 1] *= 64.0
        ref.vp[..., low, 0] = 1e-7
        ref.vp[..., low, 1] = 0.0
        w = gs * bits // 32
        ref.vc[..., low * w:(low + 1) * w] = 0
    else:
        ref.vp[..., low, :] *= 2.0 ** -apart
    cache = _cache(ref)
    cu = _cu(rows or [1] * 4)
    q = torch.randn(cu[-1], hq, d, generator=gen).to(dt)
    if rows is None:
        got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), d ** -0.5)
    else:
        got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), d ** -0.5)
    cache.check()
    _check_after_first(got, ref, q, table, lens, cu, d ** -0.5, dt)


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("hq", [8, 16])
def test_a_heavy_first_token_with_a_small_v(dt, hq):
    """The first token takes the softmax and brings a V 2^-9 of the others',
    which together bring as much: neither may be rounded away."""
    B, n, hkv, d, gs, bits = 48, 4000, 2, 128, 64, 8
    lens = [n] * B
    pages = -(-n // 64)
    gen = torch.Generator().manual_seed(42)
    ref = R.random_pool(gen, pages, 64, hkv, d, gs, bits, dt)
    table = torch.arange(pages, dtype=torch.int32)[None].expand(B, -1).contiguous()  # one prefix for all
    first = (0, slice(None), 0, 0)
    ref.kp[..., 0] *= 0.25
    ref.kp[..., 1] = (-ref.kp[..., 0].double() * 127.5).to(dt)
    ref.kp[first][..., 0] = 0.0
    ref.kp[first][..., 1] = 1.0      # logit: sum of q * scale
    ref.vp[first] = ref.vp[first] * 2.0 ** -9
    scale = 25.0 * 0.6931472 / d     # 2^25 for a q of ones
    q = (1.0 + 0.05 * torch.randn(B, hq, d, generator=gen)).to(dt)
    cache = _cache(ref)
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), scale)
    cache.check()
    want = R.attention(ref, q[:4], table[:4], lens[:4], list(range(5)), scale)
    _check(got[:4], *want, dt)


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq", [2, 4, 16])
@pytest.mark.parametrize("what", ["huge", "huge group", "inf scale", "nan scale", "inf bias"])
def test_drafts_do_not_feel_later_keys(dt, bits, hq, what):
    """The last row's own key has a V scale far above the others', or one that
    is not finite: the rows before it do not see it."""
    hkv, d, gs, n, rows = 2, 128, 64, 45, 4
    gen, ref, table = _pool(43, [n], 16, hkv, d, gs, bits, dt)
    at = _row(ref, table, 0, n - 1)
    if what == "huge":
        ref.vp[..., :] *= 2.0 ** -9
        ref.vp[at] = ref.vp[at] * (2.0 ** 20 if dt == F16 else 2.0 ** 60)
    elif what == "huge group":
        ref.vp[..., :] *= 2.0 ** -9
        # groups of neighbouring keys may lie 2^39 apart: fp16 scales always do (2^-24
        # to 2^13), 2^36 is left for bf16 next to scales that differ by up to 3
        ref.vp[at][..., 1, :] *= 2.0 ** 20 if dt == F16 else 2.0 ** 36
    else:
        ref.vp[at][..., 1, 1 if what == "inf bias" else 0] = float("nan" if what == "nan scale" else "inf")
    cache = _cache(ref)
    q = torch.randn(rows, hq, d, generator=gen).to(dt)
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32([n]), _i32([0, rows]), 0.09)
    cache.check()
    want = R.attention(ref, q[:-1], table, [n - 1], [0, rows - 1], 0.09)
    _check(got[:-1], *want, dt)
    last = R.attention(ref, q[-1:], table, [n], [0, 1], 0.09)
    if "huge" in what:
        _check(got[-1:], *last, dt)
    else:  # the group with the bad pair is not finite, the other is right
        assert not torch.isfinite(got[-1:, :, gs:]).any()
        _check(got[-1:, :, :gs], *[x[..., :gs] for x in last], dt)


@pytest.mark.parametrize("bits", [4, 8])
def test_constant_rows_near_the_largest_bf16(bits):
    """Groups of one huge value have the smallest scale and a huge bias."""
    lens, d = [300, 20], 128
    gen, ref, table = _pool(44, lens, 16, 2, d, 64, bits, BF16)
    ref.vp[..., 0] = 1e-7
    ref.vp[..., 1] = 1e37
    ref.vp[:, 1, ..., 1] *= -1.0
    cache = _cache(ref)
    q = torch.randn(2, 8, d, generator=gen).to(BF16)
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), 0.09)
    cache.check()
    _check(got, *R.attention(ref, q, table, lens, [0, 1, 2], 0.09), BF16)


def test_queries_near_the_largest_bf16():
    lens, d = [200, 64], 128
    gen, ref, table = _pool(45, lens, 16, 2, d, 64, 8, BF16)
    ref.kp *= 2.0 ** -110
    cache = _cache(ref)
    q = (1.0 + 0.3 * torch.randn(2, 8, d, generator=gen)).to(BF16) * 2.0 ** 108
    got = cache.sdpa_decode(q.cuda(), table.cuda(), _i32(lens), 0.1)
    cache.check()
    _check(got, *R.attention(ref, q, table, lens, [0, 1, 2], 0.1), BF16)


# ------------------------------------------------------------- prompt chunks --

CHUNKS = [
    # Hq, Hkv, D, gs, lens, rows, window, sinks
    (8, 2, 128, 64, [300, 90], [200, 90], 0, 0),
    (8, 2, 64, 32, [700], [260], 100, 4),
    (4, 2, 256, 64, [500, 130], [300, 130], 0, 0),
    (16, 1, 128, 128, [260], [40], 50, 0),
]


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("part", ["v", "k"])
@pytest.mark.parametrize("what", ["inf scale", "nan scale", "inf bias"])
def test_chunks_do_not_feel_hidden_keys(dt, bits, case, part, what):
    """A few keys hold a pair that is not finite.  Rows that do not see such a
    key are right; rows that do are not finite in the groups it spoils (all,
    for a K) and right in the others."""
    hq, hkv, d, gs, lens, rows, window, sinks = case
    gen, ref, table = _pool(46, lens, 16, hkv, d, gs, bits, dt)
    cu = _cu(rows)
    pairs = ref.vp if part == "v" else ref.kp
    at = {b: {n - 1, n - 7, n - r + r // 3} for b, (n, r) in enumerate(zip(lens, rows))}
    if part == "v" or window:  # before the first row: a K that all rows see would leave nothing
        at = {b: x | {max(0, lens[b] - rows[b] - 40)} for b, x in at.items()}
    at = {b: sorted(x) for b, x in at.items()}
    value = float("nan" if what == "nan scale" else "inf")
    group = {(b, j): i % (d // gs) for b in at for i, j in enumerate(at[b])}
    clean = R.RefPool(ref.pool, 16, hkv, d, gs, bits, dt)
    cpairs = clean.vp if part == "v" else clean.kp
    for (b, j), g in group.items():
        pairs[_row(ref, table, b, j)][..., g, 1 if what == "inf bias" else 0] = value
        cpairs[_row(ref, table, b, j)][..., g, :] = 0.0
    cache = _cache(ref)
    assert C.takes_chunk_kernel(cu[-1], hq, hkv, len(lens))
    q = torch.randn(cu[-1], hq, d, generator=gen).to(dt)
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), 0.09, window, sinks)
    cache.check()
    want = C.attention(clean, q, table, lens, cu, 0.09, window, sinks)
    spoilt = torch.zeros(cu[-1], 1, d, dtype=torch.bool)
    for (b, j), g in group.items():
        p = torch.arange(lens[b] - rows[b], lens[b])
        see = (j <= p) & ((window == 0) | (j > p - window) | (j < sinks))
        cols = slice(g * gs, (g + 1) * gs) if part == "v" else slice(None)
        spoilt[cu[b]:cu[b + 1], 0, cols] |= see[:, None]
    spoilt = spoilt.expand(-1, hq, -1)
    assert bool(spoilt.any()) and not bool(spoilt.all())
    assert not bool(torch.isfinite(got.cpu()[spoilt]).any())
    patched = torch.where(spoilt, want.out.to(torch.float32), got.float().cpu())
    want.check(patched, dt)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
def test_chunks_of_values_at_the_end_of_the_range(bits, d, dt):
    """Scales and biases that a row of +-the largest value gives: a code times
    the rounded scale passes the dtype's range, and counts as its end."""
    lens, rows, hkv, gs = [200, 150], [150, 149], 2, 32
    gen, ref, table = _pool(47, lens, 16, hkv, d, gs, bits, dt)
    top, last = torch.finfo(dt).max, float((1 << bits) - 1)
    s = 2 * top / last
    bump = 1.0 + 2.0 ** -7 if dt == BF16 else 1.0 + 2.0 ** -10
    ref.vp[..., 0] = torch.tensor(s * bump, dtype=torch.float64).to(dt)
    ref.vp[..., 1] = -top
    ref.kp[_row(ref, table, 0, 199)] = ref.vp[_row(ref, table, 0, 199)]  # seen by the last row alone
    cu = _cu(rows)
    k, _, v, _ = ref.rows(table[0], torch.arange(200))
    assert float(v.max()) > top * (1 + R.half_step(dt) / 2)
    cache = _cache(ref)
    q = torch.randn(cu[-1], 4, d, generator=gen).to(dt)
    got = cache.sdpa_prefill(q.cuda(), table.cuda(), _i32(lens), _i32(cu), 0.09)
    cache.check()
    want = C.attention(ref, q, table, lens, cu, 0.09)
    keep = torch.arange(cu[-1]) != 149
    for n in ("out", "mag", "sq", "l1", "keys"):
        setattr(want, n, getattr(want, n)[keep])
    want.check(got[keep.cuda()], dt)


# ----------------------------------------------------- what nobody is to see --

HIDDEN = [
    # Hq, Hkv, D, gs, lens, rows (None: single tokens), window, sinks
    (8, 2, 128, 64, [1000, 17, 333, 5], None, 0, 0),
    (16, 2, 128, 32, [700, 33], None, 100, 3),
    (16, 1, 64, 32, [555, 70], None, 0, 0),
    (8, 2, 256, 64, [300, 41], None, 50, 0),
    (8, 2, 128, 64, [200, 90], [5, 3], 40, 2),
    (8, 2, 128, 64, [400, 190], [300, 130], 100, 5),
    (4, 2, 256, 32, [500, 100], [200, 100], 0, 0),
    # enough for a warp to meet several tiles of a sequence
    (32, 8, 128, 64, [300 + 37 * i % 600 for i in range(56)], None, 0, 0),
    (64, 8, 64, 32, [300 + 37 * i % 600 for i in range(56)], None, 0, 0),
    (16, 8, 128, 32, [300 + 37 * i % 600 for i in range(56)], [1 + i % 5 for i in range(56)], 150, 2),
]


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", HIDDEN, ids=lambda c: "-".join(str(x) for x in c)[:48])
def test_rows_that_nobody_sees_do_not_change_a_bit(dt, bits, case):
    """The rows behind a sequence's end, and those that its window has left, hold
    zeros, ordinary, huge or no numbers."""
    hq, hkv, d, gs, lens, rows, window, sinks = case
    gen, ref, table = _pool(48, lens, 16, hkv, d, gs, bits, dt)
    seen = torch.zeros(ref.kc.shape[0], ref.kc.shape[2], 16, dtype=torch.bool)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        first = n - (1 if rows is None else rows[b])
        keep = j[(j < sinks) | (j > first - window)] if window else j
        seen[ref.index(table[b], keep)] = True
    hidden = ~seen[:, None, :, :, None, None]
    cu = _cu(rows or [1] * len(lens))
    q = torch.randn(cu[-1], hq, d, generator=gen).to(dt).cuda()
    results = []
    for what in (0.0, 1.0, -1.0, torch.finfo(dt).max, float("inf"), float("nan")):
        other = R.RefPool(ref.pool, 16, hkv, d, gs, bits, dt)
        for p in (other.kp, other.vp):
            p.copy_(torch.where(hidden.expand_as(p), torch.full_like(p, what), p))
        cache = _cache(other)
        for _ in range(2):
            if rows is None:
                got = cache.sdpa_decode(q, table.cuda(), _i32(lens), 0.1, window, sinks)
            else:
                got = cache.sdpa_prefill(q, table.cuda(), _i32(lens), _i32(cu), 0.1, window, sinks)
            results.append(got.view(torch.int16).cpu())
        cache.check()
    assert all(torch.equal(r, results[0]) for r in results)
