"""Ragged chunk attention on the GPU, held to what the chunk kernel's chosen
roundings leave (tests/paged_chunk_ref.py)."""
import numpy as np
import pytest
import torch

import paged_chunk_ref as C
import paged_ref as R
from test_gpu_paged import PREFILL, _cache, _check, _cu, _i32, _pages

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16

MORE = [
    # dt, bits, gs, Hq, Hkv, D, page, lens, rows, pad, window, sinks
    (BF16, 8, 64, 8, 1, 128, 64, [1500], [300], 0, 0, 0),
    (BF16, 8, 32, 16, 2, 64, 16, [900, 333], [200, 333], 3, 200, 17),
    (BF16, 4, 32, 12, 2, 64, 32, [700], [150], 0, 0, 0),
    (F16, 4, 128, 16, 2, 128, 256, [1111], [222], 0, 300, 1),
    (F16, 8, 128, 8, 2, 256, 64, [800, 100], [300, 100], 0, 0, 0),
    (BF16, 8, 32, 10, 2, 256, 16, [500], [129], 1, 100, 33),
    (BF16, 4, 64, 8, 8, 256, 128, [640], [256], 0, 0, 0),
    (F16, 4, 32, 6, 2, 256, 32, [333, 65], [120, 65], 0, 64, 0),
    (F16, 8, 64, 2, 2, 64, 16, [4000], [1000], 0, 0, 0),
]


@pytest.mark.parametrize("case", PREFILL + MORE, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("form", ["plain", "strided q, negative scale"])
def test_prefill_roundings(case, form):
    dt, bits, gs, hq, hkv, d, page, lens, rows, pad, window, sinks = case
    gen = torch.Generator().manual_seed(12)
    pages = _pages(lens, page)
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, pages)
    R.poison(ref, table, lens)
    cache = _cache(ref)
    cu, scale = _cu(rows), d ** -0.5
    T = cu[-1] + pad
    if form == "plain":
        q = torch.randn(T, hq, d, generator=gen).to(dt).cuda()
    else:  # heads of a wider projection, at an odd element
        scale = -scale
        q = torch.randn(T, (hq + 2) * d + 3, generator=gen).to(dt).cuda()[:, 1:-2]
        q = q.unflatten(1, (hq + 2, d))[:, 1:1 + hq]
        assert not q.is_contiguous() and q.data_ptr() % 16
    got = cache.sdpa_prefill(q, table.cuda(), _i32(lens), _i32(cu), scale, window, sinks)[:cu[-1]]
    cache.check()
    q = q.cpu()[:cu[-1]]
    if C.takes_chunk_kernel(T, hq, hkv, len(lens)):
        C.attention(ref, q, table, lens, cu, scale, window, sinks).check(got, dt)
    else:
        out, mag, magc, l1 = R.attention(ref, q, table, lens, cu, scale, window, sinks)
        _check(got, out, mag, magc, l1.abs(), dt)


@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_heavy_first_token_leaves_the_others_their_share(dt, bits, d):
    """The first token takes nearly all of the softmax and brings nothing (v =
    0); what the others bring, each with 2^-25.4 of its probability, is the whole
    output.  Known in closed form: every other logit is 0 and every other v 1."""
    hkv, hq, page, gs, n, rows = 8, 32, 64, 32, 16000, 1536
    pages = n // page
    ref = R.random_pool(torch.Generator().manual_seed(1), pages, page, hkv, d, gs, bits, dt)
    ref.kp.zero_()
    ref.vp.zero_()
    ref.vp[..., 1] = 1.0
    table = torch.arange(pages, dtype=torch.int32)[None]
    # q is 1 in every element: the first key's logit is sum k * scale
    ref.vp[0, :, 0, 0] = 0.0
    k0 = 1.0
    ref.kp[0, :, 0, 0, :, 1] = k0
    x = 25.4 * float(np.log(2.0))
    scale = x / (k0 * d)
    cache = _cache(ref)
    q = torch.ones(rows, hq, d, dtype=dt, device="cuda")
    got = cache.sdpa_prefill(q, table.cuda(), _i32([n]), _i32([0, rows]), scale)
    cache.check()
    others = torch.arange(n - rows, n, dtype=torch.float64)
    e = 2.0 ** -25.4
    want = (others * e / (1 + others * e))[:, None, None]
    # a probability's half step, fp16's subnormal steps of 2^-32 for each key, the
    # logit (2^-18 of its 25 for the f32 sum, and 2^-24 of it for the scale), the output
    u = R.half_step(dt)
    tol = 2 * u * want + (others * 2.0 ** -32)[:, None, None] * (dt == F16) + 2 * (2.0 ** -18 * x) * want + \
        (3e-8 if dt == F16 else 0)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
