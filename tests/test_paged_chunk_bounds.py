"""The bounds that the chunk kernel's results are held to reject wrong results:
mistakes planted in the 64-bit reference, on the CPU, for every prompt-chunk
case that the GPU tests run through that kernel."""
import numpy as np
import pytest
import torch

import paged_chunk_ref as C
import paged_ref as R
from test_gpu_paged import PREFILL

CASES = [c for c in PREFILL if C.takes_chunk_kernel(sum(c[8]) + c[9], c[3], c[4], len(c[7]))]


def _setup(case):
    dt, bits, gs, hq, hkv, d, page, lens, rows, pad, window, sinks = case
    gen = torch.Generator().manual_seed(12)
    pages = sum(-(-n // page) for n in lens) + 3
    ref = R.random_pool(gen, pages, page, hkv, d, gs, bits, dt)
    table = R.make_table(gen, lens, page, pages)
    cu = [0] + list(np.cumsum(rows))
    q = torch.randn(cu[-1], hq, d, generator=gen).to(dt)
    return ref, q, table, lens, cu, d ** -0.5, window, sinks


def _code_up(ref, keys):
    """The pool with every code of K (or V) one up."""
    other = R.RefPool(ref.pool, ref.page, ref.heads, ref.d, ref.gs, ref.bits, ref.dt)
    words = other.kc if keys else other.vc
    mask = (1 << ref.bits) - 1
    out = torch.zeros_like(words)
    for s in range(0, 32, ref.bits):
        out |= (((words >> s) & mask) + 1).clamp_max(mask) << s
    words.copy_(out)
    return other


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_wrong_results_fail(case):
    ref, q, table, lens, cu, scale, window, sinks = _setup(case)
    dt = ref.dt
    want = C.attention(ref, q, table, lens, cu, scale, window, sinks)
    want.check(want.out.float().to(dt), dt)

    def seen(change):
        def f(qpos, n, window, sinks):
            return change(torch.arange(n)[None], qpos, C.visible(qpos, n, window, sinks))
        return f

    bad = {
        "zeros": lambda: 0 * want.out,
        "no q k": lambda: C.attention(ref, q, table, lens, cu, 0.0, window, sinks).out,
        "scale": lambda: C.attention(ref, q, table, lens, cu, 0.9 * scale, window, sinks).out,
        "k codes": lambda: C.attention(_code_up(ref, True), q, table, lens, cu, scale, window, sinks).out,
        "v codes": lambda: C.attention(_code_up(ref, False), q, table, lens, cu, scale, window, sinks).out,
        "one key more": lambda: C.attention(ref, q, table, lens, cu, scale, window, sinks, see_fn=seen(
            lambda j, p, see: see | (j == p + 1))).out,
        "last key lost": lambda: C.attention(ref, q, table, lens, cu, scale, window, sinks, see_fn=seen(
            lambda j, p, see: see & (j != p))).out,
        "tile lost": lambda: C.attention(ref, q, table, lens, cu, scale, window, sinks, see_fn=seen(
            lambda j, p, see: see & ((j >> 4) != 2) if window == 0 else see & ((j >> 4) != (p >> 4) - 1))).out,
    }
    if window:
        bad["window + 1"] = lambda: C.attention(ref, q, table, lens, cu, scale, window + 1, sinks).out
        if window > 1:
            bad["window - 1"] = lambda: C.attention(ref, q, table, lens, cu, scale, window - 1, sinks).out
        if sinks:
            bad["sink lost"] = lambda: C.attention(ref, q, table, lens, cu, scale, window, sinks - 1).out
    if 0 < window < 32:
        del bad["tile lost"]  # hardly any row has that tile in its window
    accepted = []
    for name, wrong in bad.items():
        try:
            want.check(wrong().float().to(dt), dt)
            accepted.append(name)
        except AssertionError:
            pass
    assert not accepted


def test_rounding_to_the_dtype():
    x = torch.randn(4096, dtype=torch.float64) * torch.exp2(torch.randint(-30, 14, (4096,)).double())
    for dt in (torch.float16, torch.bfloat16):
        y = x.to(dt).double()  # through f32: equal but for its rare double roundings
        z = C.round_to(x, dt)
        assert float((y != z).double().mean()) < 1e-3
        assert bool(((z - x).abs() <= (y - x).abs()).all())
        big = torch.tensor([7e38, -7e38], dtype=torch.float64)
        top = torch.finfo(dt).max
        assert C.round_to(big, dt).tolist() == [top, -top]
