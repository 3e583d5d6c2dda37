"""What the paged cache's chunk kernel computes, in 64 bits with its chosen
roundings put in, and how far it may be from that.

sdpa_prefill takes the chunk kernel when rows * (heads of a group) pass 64 times
the sequences, rows counting the whole buffer; it holds K and V rounded to the
dtype, as a dense cache would, and clamped to its range.  That rounding is
reproduced here exactly (code * scale + bias is exact in 64 bits), so what is
left to allow for is

  * the probabilities, rounded to the dtype: p_j (1 + d_j), |d_j| <= u, half a
    step of the dtype; fp16's below 2^-14 of the 2^7 that the largest stands
    for are subnormal, off by at most 2^-25 / 2^7 = 2^-32 of it;
  * logits summed in f32: 2^-18 of sum |q| |k| (as for the column kernel), and
    ex2's 2^-20, above and below the line; the output's f32 sums, one addition
    for every 16 keys, each off by at most 2^-23 of sum p |v|;
  * the output, rounded once: u of it.

Elementwise the worst case of their sum is allowed.  It is far above what
happens, since the d_j of different keys are independent: over a case, the
root mean square of the error is held to 1.5 times that of its parts, with
|d| <= u uniform (variance u^2 / 3 at most) for each p_j and for the output,
and the f32 part at its worst case.  1.5: the mean over mantissas of a
rounding's relative variance is only half of u^2 / 3, so a sound kernel stays
near 0.7 and twice the expected error does not pass."""
from __future__ import annotations

import math

import torch

import paged_ref as R

BITS = {torch.float16: 11, torch.bfloat16: 8}   # significant bits


def takes_chunk_kernel(rows, hq, hkv, batch):
    return rows * (hq // hkv) > 64 * batch


def round_to(x, dt):
    """f64 values to the nearest of the dtype (ties to even), clamped."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - BITS[dt]).clamp_min(-24 if dt == torch.float16 else -133))
    top = torch.finfo(dt).max
    return (torch.round(x / step) * step).clamp(-top, top)


class Want:
    """Exact outputs of the rounded cache, and their error terms per element."""

    def __init__(self, T, hq, d):
        z = lambda n: torch.zeros(T, hq, n, dtype=torch.float64)
        self.out, self.mag, self.sq, self.l1, self.keys = z(d), z(d), z(d), z(1), z(1)
        self.vmax = 0.0

    def _f32(self):
        return (2 * (2.0 ** -18 * self.l1 + 2.0 ** -20) + 2.0 ** -27 * self.keys) * self.mag

    def check(self, got, dt):
        """Raises when `got` is further away than the bounds above."""
        u = R.half_step(dt)
        d = (got.double().cpu() - self.out).abs()
        assert bool(torch.isfinite(d).all()), "not finite"
        tiny = 2.0 ** -32 * self.keys * self.vmax if dt == torch.float16 else 0.0
        err = u * self.mag + self._f32() + tiny
        floor = 3e-8 if dt == torch.float16 else 0.0
        tol = u * (self.out.abs() + err) + err + floor
        bad = d > tol
        assert not bool(bad.any()), f"{int(bad.sum())} outside, up to {float((d / tol).max()):.3f} times"
        var = u * u / 3 * (self.sq + self.out ** 2) + (self._f32() + tiny + floor) ** 2
        rms, want = math.sqrt(float((d ** 2).mean())), math.sqrt(float(var.mean()))
        assert rms <= 1.5 * want, f"rms {rms:.3e}, {rms / want:.2f} times the roundings' own"


def visible(qpos, n, window, sinks):
    j = torch.arange(n)[None]
    see = j <= qpos
    if window > 0:
        see &= (j > qpos - window) | (j < sinks)
    return see


def attention(ref, q, table, lens, cu, scale, window=0, sinks=0, dense=True, see_fn=visible):
    """dense: K and V rounded to the dtype.  see_fn: for planted mistakes."""
    T, hq, d = q.shape
    rep, dt = hq // ref.heads, ref.dt
    w = Want(T, hq, d)
    qd = q.double()
    for b, n in enumerate(lens):
        r0, r1 = cu[b], cu[b + 1]
        if r1 <= r0 or n <= 0:
            continue
        k, _, v, _ = ref.rows(table[b], torch.arange(n))
        if dense:
            k, v = round_to(k, dt), round_to(v, dt)
        w.vmax = max(w.vmax, float(v.abs().max()))
        qpos = torch.arange(n - (r1 - r0), n)[:, None]
        see = see_fn(qpos, n, window, sinks)
        some = see.any(1)
        for g in range(ref.heads):
            kk, vv = k[:, g], v[:, g]
            h = slice(g * rep, (g + 1) * rep)
            x = qd[r0:r1, h]                                   # [rows, rep, d]
            s = (x.flatten(0, 1) @ kk.T * scale).unflatten(0, (r1 - r0, rep))
            s = s.masked_fill(~see[:, None], float("-inf"))
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isfinite(m), m, 0.0))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            p[~some] = 0
            p = p.flatten(0, 1)
            put = lambda dst, y: dst[r0:r1, h].copy_(y.unflatten(0, (r1 - r0, rep)))
            put(w.out, p @ vv)
            put(w.mag, p @ vv.abs())
            put(w.sq, (p * p) @ (vv * vv))
            a = (x.flatten(0, 1).abs() @ kk.abs().T * abs(scale)).unflatten(0, (r1 - r0, rep))
            put(w.l1, a.masked_fill(~see[:, None], 0.0).amax(-1, keepdim=True).flatten(0, 1))
            put(w.keys, see.sum(1).double()[:, None, None].expand(-1, rep, 1).flatten(0, 1))
    return w
