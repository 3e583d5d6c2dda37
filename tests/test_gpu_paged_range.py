"""Attention over pages whose scales lie far apart, or are not finite where a
query does not look, on the GPU against the plain 64-bit implementation."""
import pytest
import torch

import paged_chunk_ref as C
import paged_ref as R
from test_gpu_paged import _cache, _cu, _i32, _pages

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
