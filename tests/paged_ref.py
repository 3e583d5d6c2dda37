"""A plain 64-bit implementation of the paged cache's operators on the CPU,
from their definitions, for the tests."""
from __future__ import annotations

import numpy as np
import torch

from oracle import oracle as O

TILE = 16
U16 = 2.0 ** -11  # half a step of fp16, relative


def half_step(dt):
    return torch.finfo(dt).eps / 2


class RefPool:
    """Host copy of a pool with its parts as views."""

    def __init__(self, pool, page, heads, d, gs, bits, dt):
        self.pool = pool.cpu().clone()
        self.page, self.heads, self.d, self.gs, self.bits, self.dt = page, heads, d, gs, bits, dt
        w, g = d * bits // 32, d // gs
        self.w, self.g, o, parts = w, g, 0, []
        for _ in range(2):
            parts.append(self.pool[..., o:o + TILE * w].unflatten(-1, (TILE, w)))
            o += TILE * w
            pr = self.pool[..., o:o + TILE * g].unflatten(-1, (TILE, g))
            parts.append(pr.view(dt).unflatten(-1, (g, 2)))
            o += TILE * g
        assert o == self.pool.shape[-1]
        self.kc, self.kp, self.vc, self.vp = parts

    def index(self, table, pos):
        pos = torch.as_tensor(pos)
        return table[pos // self.page].long(), (pos % self.page) // TILE, pos % TILE

    def rows(self, table, pos):
        """K and V at positions `pos` of one sequence, f64 [n, heads, d], and
        what their rounding errors go by: |s| c + |z| of K and |s| max(c, top -
        c) of V, for v = s c + z with codes up to `top`."""
        pg, tile, row = self.index(table, pos)
        shift = torch.arange(0, 32, self.bits, dtype=torch.int32)
        out, top = [], float((1 << self.bits) - 1)
        for codes, pairs in ((self.kc, self.kp), (self.vc, self.vp)):
            c = (codes[pg, :, tile, row][..., None] >> shift) & ((1 << self.bits) - 1)
            c = c.flatten(-2).double().unflatten(-1, (self.g, self.gs))
            p = pairs[pg, :, tile, row].double()
            a = p[..., :1].abs()
            out.append((c * p[..., :1] + p[..., 1:]).flatten(-2))
            out.append((a * c + p[..., 1:].abs() if len(out) < 2 else
                        a * torch.maximum(c, top - c)).flatten(-2))
        return out

    def put(self, table, pos, k, v):
        """Quantize rows k, v [n, heads, d] (dtype, k rotated) with the oracle
        and write them."""
        pg, tile, row = self.index(table, pos)
        odt = O.F16 if self.dt == torch.float16 else O.BF16
        for x, codes, pairs in ((k, self.kc, self.kp), (v, self.vc, self.vp)):
            n = x.shape[0]
            bits16 = x.contiguous().view(torch.int16).numpy().view(np.uint16)
            c, s, z = O.quantize(bits16[None], self.gs, self.bits, odt)
            codes[pg, :, tile, row] = torch.from_numpy(c[0].view(np.int32).reshape(n, -1, self.w))
            sz = torch.stack([torch.from_numpy(t[0].view(np.int16).reshape(n, -1, self.g))
                              for t in (s, z)], -1)
            pairs[pg, :, tile, row] = sz.view(self.dt)


def rotate(x, pos, dims, base=10000.0, scale=1.0, traditional=False, freqs=None, pre=1.0):
    """x [n, heads, d] dtype at positions pos [n]: 64-bit rotation, rounded to
    32 bits and then to the dtype."""
    if not dims:
        return x
    i = torch.arange(dims // 2, dtype=torch.float64)
    inv = 1.0 / freqs.double() if freqs is not None else \
        float(np.float32(base)) ** (-2.0 * i / dims)
    ang = (float(np.float32(scale)) * torch.as_tensor(pos).double())[:, None, None] * inv
    pre = float(np.float32(pre))
    c, s = torch.cos(ang) * pre, torch.sin(ang) * pre
    y = x.double()
    out = y.clone()
    if traditional:
        a, b = y[..., 0:dims:2], y[..., 1:dims:2]
        out[..., 0:dims:2], out[..., 1:dims:2] = a * c - b * s, a * s + b * c
    else:
        a, b = y[..., :dims // 2], y[..., dims // 2:dims]
        out[..., :dims // 2], out[..., dims // 2:dims] = a * c - b * s, a * s + b * c
    return out.float().to(x.dtype)


def attention(ref, q, table, lens, cu, scale, window=0, sinks=0):
    """f64 outputs [rows, heads, d] and the magnitudes that the tolerance
    counts: sum_j p_j |v_j| and sum_j p_j |s_j| max(c_j, top - c_j) per
    element, and the largest sum_d |q_d| (|s| c + |z|)_jd * scale over the
    visible keys per row and head."""
    T, Hq, d = q.shape
    rep = Hq // ref.heads
    out = torch.zeros(T, Hq, d, dtype=torch.float64)
    mag, magc = torch.zeros_like(out), torch.zeros_like(out)
    l1 = torch.zeros(T, Hq, 1, dtype=torch.float64)
    q = q.double()
    for b, n in enumerate(lens):
        r0, r1 = cu[b], cu[b + 1]
        if r1 <= r0 or n <= 0:
            continue
        k, ka, v, va = ref.rows(table[b], torch.arange(n))
        qpos = torch.arange(n - (r1 - r0), n)[:, None]
        j = torch.arange(n)[None]
        see = j <= qpos
        if window > 0:
            see &= (j > qpos - window) | (j < sinks)
        for h in range(Hq):
            g = h // rep
            s = (q[r0:r1, h] @ k[:, g].T * scale).masked_fill(~see, float("-inf"))
            some = see.any(1)
            e = torch.exp(s - s.amax(1, keepdim=True).nan_to_num(neginf=0.0))
            p = torch.where(see, e, 0.0) / e.sum(1, keepdim=True).clamp_min(1e-300)
            p[~some] = 0
            out[r0:r1, h] = p @ v[:, g]
            mag[r0:r1, h] = p @ v[:, g].abs()
            magc[r0:r1, h] = p @ va[:, g]
            a = (q[r0:r1, h].abs() @ ka[:, g].T * scale).masked_fill(~see, 0.0)
            l1[r0:r1, h] = a.amax(1, keepdim=True)
    return out, mag, magc, l1


def tolerance(out, mag, magc, l1, dt, dense):
    """How far a kernel may be from the exact output.

    Every output is rounded once: half a step of it.  Probabilities carry the
    error of a logit summed in f32 over scales times codes, taken as 2^-18 of
    sum |q| (|s| c + |z|) (16 partial sums and the two folds are some 20
    roundings of 2^-24; 2^-18 is three times that), and ex2's 2^-20; it enters
    the sums above and below the line: 2 of them, times sum p |v|.

    The column kernel rounds p s to fp16, which multiplies c (bf16 outputs) or
    c minus the middle code (fp16 outputs); both are at most max(c, top - c):
    half a step of fp16, and 2^-18 for the f32 sums of s c + z, of magc.

    dense: the chunk kernel may have run instead, which rounds p, K and V to
    the dtype before their products: two half steps of sum p |v|, and one of
    the logit's sum."""
    u = half_step(dt) if dense else 0.0
    p = (2.0 ** -18 + u) * l1 + 2.0 ** -20
    err = (2 * p + 2 * u) * mag + (U16 + 2.0 ** -18) * magc
    floor = 3e-8 if dt == torch.float16 else 0.0  # half of fp16's subnormal step
    return half_step(dt) * (out.abs() + err) + err + floor


def random_pool(gen, pages, page, heads, d, gs, bits, dt):
    """A pool of random codes with scales and biases of both signs."""
    w, g = d * bits // 32, d // gs
    pool = torch.randint(-2 ** 31, 2 ** 31, (pages, heads, page // TILE, 2 * TILE * (w + g)),
                         generator=gen, dtype=torch.int64).to(torch.int32)
    ref = RefPool(pool, page, heads, d, gs, bits, dt)
    for p in (ref.kp, ref.vp):
        s = (torch.rand(p.shape[:-1], generator=gen) + 0.5) * (4.0 / (1 << bits))
        s *= torch.where(torch.rand(s.shape, generator=gen) < 0.5, -1.0, 1.0)
        mid = -s * ((1 << bits) - 1) / 2
        p[..., 0] = s.to(dt)
        p[..., 1] = (mid + 0.2 * torch.randn(s.shape, generator=gen)).to(dt)
    return ref


def poison(ref, table, lens):
    """NaN and infinite scales in every row that no sequence owns."""
    own = torch.zeros(ref.kc.shape[0], ref.kc.shape[2], TILE, dtype=torch.bool)
    for b, n in enumerate(lens):
        if n > 0:
            pg, tile, row = ref.index(table[b], torch.arange(n))
            own[pg, tile, row] = True
    for p in (ref.kp, ref.vp):
        bad = torch.where(torch.rand(p.shape) < 0.5, float("nan"), float("inf")).to(p.dtype)
        keep = own[:, None, :, :, None, None].expand_as(p)
        p.copy_(torch.where(keep, p, bad))


def make_table(gen, lens, page, pages, extra=2, unused=2 ** 31 - 1):
    """A shuffled page table; entries behind a sequence's last page hold a
    number outside the pool."""
    need = [-(-max(n, 0) // page) for n in lens]
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + extra), unused, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table
