"""The paged quantized KV cache's operators, measured: append (RoPE + quantize
+ write into pages), single-token attention and chunk attention over the pages.

A pool is an int32 tensor [pages, kv_heads, page_size / 16, tile_words].  One
tile holds 16 consecutive token rows of one kv head:

    K codes [16][D * bits / 32] words, K (scale, bias) pairs [16][D / group]
    words (scale in the low half), then V codes and V pairs laid out the same.

Token position p of sequence b lies in page page_table[b][p // page_size],
tile (p % page_size) // 16, row p % 16.  seq_lens counts the tokens of each
sequence with this step's rows included: row j of the n rows that sequence b
brings stands at position seq_lens[b] - n + j.  cu_rows holds the sequences'
first rows; rows behind cu_rows[B] are padding and stay as they were.

Definitions:
  append     angle = (rope_scale * position) * inv_freq in 64 bits, K (and Q)
             rotated in 64 bits and rounded to 32 and then to the tensor's
             type; the rows' groups quantized by the affine rule in 32-bit
             IEEE steps (the codes are defined by those steps, bit for bit).
  attention  softmax(scale * q . k) v over the visible keys with k, v = code *
             scale + bias, unrounded; query position p sees key j when j <= p
             and (window == 0 or j > p - window or j < sinks); a row that
             sees nothing gives zeros.

`own` false: plain torch in 32 bits (64 for the rotation).  `own` true: the
calls of the framework's paged cache.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
TILE = 16
QUANT_EPS = 1e-7


# ---------------------------------------------------------------- the cases --

def listed():
    return [
        # One user's decode step, the layer shape of the single-sequence decode
        # configuration: a call of a few microseconds where latency is all.
        dict(name="append-1-row", op="append", dtype="fp16", bits=8, gs=64, hq=16, hkv=4, d=128,
             page=64, batch=1, min_len=2048, max_len=2048, min_rows=1, max_rows=1, pad=0,
             rope_dims=128, base=10000.0, table=False, traditional=False, lens_seed=1),
        # A serving step: one new row for each of 64 sequences at different
        # lengths, 4-bit pages.
        dict(name="append-64-rows", op="append", dtype="bf16", bits=4, gs=64, hq=32, hkv=8, d=128,
             page=16, batch=64, min_len=64, max_len=4096, min_rows=1, max_rows=1, pad=0,
             rope_dims=128, base=500000.0, table=False, traditional=False, lens_seed=2),
        # Prompt chunks of several requests batched together (Gemma-4-12B's
        # sliding layer: 16 query and 8 kv heads of 256), partial rotation by a
        # frequency table, a few padding rows at the end.
        dict(name="append-chunks", op="append", dtype="bf16", bits=8, gs=64, hq=16, hkv=8, d=256,
             page=32, batch=5, min_len=1500, max_len=9000, min_rows=900, max_rows=2300, pad=13,
             rope_dims=128, base=10000.0, table=True, traditional=False, lens_seed=3),
        # Decode of one sequence, 2048 keys in 8 bits.
        dict(name="decode-2048", op="decode", dtype="fp16", bits=8, gs=64, hq=16, hkv=4, d=128,
             page=64, batch=1, min_len=2048, max_len=2048, window=0, sinks=0, lens_seed=4),
        # Batched 4-bit decode, 8 sequences of 8193 keys, small pages.
        dict(name="decode-8x8193", op="decode", dtype="fp16", bits=4, gs=64, hq=32, hkv=8, d=128,
             page=16, batch=8, min_len=8193, max_len=8193, window=0, sinks=0, lens_seed=5),
        # Sliding-window layer with the first tokens kept visible, head size 256.
        dict(name="decode-window-d256", op="decode", dtype="bf16", bits=8, gs=64, hq=8, hkv=4,
             d=256, page=32, batch=4, min_len=3000, max_len=4096, window=1024, sinks=4,
             lens_seed=6),
        # Long-context serving: 64 ragged sequences of up to 32768 keys, 4 bits.
        dict(name="decode-64-ragged", op="decode", dtype="fp16", bits=4, gs=64, hq=32, hkv=8,
             d=128, page=64, batch=64, min_len=1024, max_len=32768, window=0, sinks=0,
             lens_seed=7),
        # The same batch through a layer that sees 4096 keys and 16 sinks.
        dict(name="decode-64-window", op="decode", dtype="bf16", bits=4, gs=64, hq=32, hkv=8,
             d=128, page=16, batch=64, min_len=1024, max_len=32768, window=4096, sinks=16,
             lens_seed=8),
        # A step that checks 1 to 8 drafted tokens for each of 16 sequences.
        dict(name="prefill-drafts", op="prefill", dtype="fp16", bits=4, gs=64, hq=32, hkv=8,
             d=128, page=16, batch=16, min_len=512, max_len=8192, min_rows=1, max_rows=8, pad=3,
             window=0, sinks=0, lens_seed=9),
        # A 512-token chunk over a 16384-token cache in 8 bits.
        dict(name="prefill-512-of-16896", op="prefill", dtype="fp16", bits=8, gs=64, hq=32, hkv=8,
             d=128, page=64, batch=1, min_len=16896, max_len=16896, min_rows=512, max_rows=512,
             pad=0, window=0, sinks=0, lens_seed=10),
        # Ragged chunks of a batch, 4 bits, a window with sinks.
        dict(name="prefill-ragged-window", op="prefill", dtype="bf16", bits=4, gs=64, hq=32, hkv=8,
             d=128, page=16, batch=6, min_len=2500, max_len=16384, min_rows=1, max_rows=2000,
             pad=9, window=1024, sinks=4, lens_seed=11),
        # A prompt chunk through a sliding layer of Gemma-4-12B's shape.
        dict(name="prefill-window-d256", op="prefill", dtype="bf16", bits=8, gs=64, hq=16, hkv=8,
             d=256, page=32, batch=2, min_len=1500, max_len=5000, min_rows=700, max_rows=1024,
             pad=0, window=1024, sinks=0, lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: types, widths, head layouts, pages and lengths over the
    whole range, none costlier than the largest listed one of its kind."""
    op = rng.choice(["append", "decode", "prefill"])
    d = rng.choice([64, 128, 256])
    gs = rng.choice([g for g in (32, 64, 128) if g <= d])
    hkv = rng.choice([1, 2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 5, 8, 16])
    while hkv * rep * d > 8192:
        rep = rng.choice([1, 2, 4])
    c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]), bits=rng.choice([4, 8]), gs=gs,
             hq=hkv * rep, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 128]),
             lens_seed=rng.randrange(1 << 30))
    if op == "append":
        c["batch"] = _log_int(rng, 1, 128)
        c["max_rows"] = 1 if rng.random() < 0.4 else _log_int(rng, 1, 8192 // c["batch"])
        c["min_rows"] = 1 if rng.random() < 0.5 else max(1, c["max_rows"] // 2)
        c["max_len"] = max(c["max_rows"], _log_int(rng, 16, 131072 // c["batch"]))
        c["min_len"] = max(c["max_rows"], c["max_len"] // 3)
        c["pad"] = rng.choice([0, 1, 7])
        c["rope_dims"] = rng.choice([0, d // 2, d, d])
        c["base"] = rng.choice([10000.0, 500000.0, 1000000.0])
        c["table"] = rng.random() < 0.5
        c["traditional"] = rng.random() < 0.3
    elif op == "decode":
        c["batch"] = _log_int(rng, 1, 200)
        tokens = (1 << 30) // (hkv * d)
        c["max_len"] = _log_int(rng, 16, max(32, min(131072, tokens // c["batch"])))
        c["min_len"] = rng.choice([1, max(1, c["max_len"] // 3), c["max_len"]])
    else:
        c["batch"] = _log_int(rng, 1, 24)
        c["max_len"] = _log_int(rng, 32, 16896)
        rows = int(1.3e11 / (4.0 * c["hq"] * d * c["max_len"] * c["batch"]))
        c["max_rows"] = _log_int(rng, 1, max(1, min(rows, c["max_len"], 2048)))
        c["min_rows"] = rng.choice([1, max(1, c["max_rows"] // 2)])
        c["min_len"] = max(c["max_rows"], c["max_len"] // 3)
        c["pad"] = rng.choice([0, 5])
    if op != "append":
        if rng.random() < 0.5:
            c["window"], c["sinks"] = 0, 0
        else:
            c["window"] = _log_int(rng, 1, max(2, c["max_len"]))
            c["sinks"] = rng.choice([0, 1, 4, 20])
    return c


def _shape(case):
    """The lengths and row counts of the case's sequences (host lists)."""
    r = random.Random(case["lens_seed"])
    lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]
    if case["op"] == "decode":
        return lens, [1] * case["batch"]
    return lens, [r.randint(case["min_rows"], case["max_rows"]) for _ in range(case["batch"])]


def _row_words(case):
    """Words of one K (or V) row in a tile: codes, and scale / bias pairs."""
    return case["d"] * case["bits"] // 32, case["d"] // case["gs"]


def _visible(pos, window, sinks):
    """Keys that the query at `pos` sees."""
    if window <= 0:
        return pos + 1
    lo = max(0, pos - window + 1)
    return pos + 1 - lo + min(max(sinks, 0), lo)


def work(case):
    lens, rows = _shape(case)
    w, g = _row_words(case)
    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    kv_row = 2 * 4 * (w + g) * hkv  # bytes of a token's K and V in the pages
    total = sum(rows)
    if case["op"] == "append":
        # read q, k, v; write q and the token's K / V rows
        nbytes = total * (2 * d * (2 * hq + 2 * hkv) + kv_row)
        flops = total * (3 * case["rope_dims"] * (hq + hkv) + 2 * hkv * d * 6)
        return {"bytes": nbytes, "flops": flops}
    window, sinks = case["window"], case["sinks"]
    keys = pairs = 0
    for n, r in zip(lens, rows):
        first = n - r
        lo = max(0, first - window + 1) if window > 0 else 0
        keys += n - lo + min(max(sinks, 0), lo)
        pairs += sum(_visible(p, window, sinks) for p in range(first, n))
    nbytes = keys * kv_row + 2 * total * hq * d * 2
    return {"bytes": nbytes, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------- preparation --

def _torch_dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _components(pool, case):
    """K codes, K pairs, V codes, V pairs as views of the pool: codes int32
    [P, H, T, 16, words], pairs [P, H, T, 16, groups, 2] in the dtype."""
    w, g = _row_words(case)
    dt = _torch_dtype(case)
    out, o = [], 0
    for _ in range(2):
        out.append(pool[..., o:o + TILE * w].unflatten(-1, (TILE, w)))
        o += TILE * w
        out.append(pool[..., o:o + TILE * g].unflatten(-1, (TILE, g)).view(dt).unflatten(-1, (g, 2)))
        o += TILE * g
    return out


def _round_away(x):
    t = torch.trunc(x)
    return t + torch.where((x - t).abs() >= 0.5, torch.sign(x), torch.zeros_like(x))


def _quantise(x, bits, gs):
    """The affine group rule on f32 values [..., D]: int32 codes, scales and
    biases in f32.  Divisors are tensors, so that they are IEEE divisions."""
    xg = x.unflatten(-1, (-1, gs))
    mn, mx = xg.amin(-1), xg.amax(-1)
    s0 = (mx - mn) / torch.full_like(mx, float((1 << bits) - 1))
    s0 = torch.where(s0 >= QUANT_EPS, s0, torch.full_like(s0, QUANT_EPS))
    neg = mn.abs() > mx.abs()
    anchor = torch.where(neg, mn, mx)
    s0 = torch.where(neg, s0, -s0)
    q0 = _round_away(anchor / s0)
    some = q0 != 0
    scale = torch.where(some, anchor / torch.where(some, q0, torch.ones_like(q0)), s0)
    bias = torch.where(some, anchor, torch.zeros_like(anchor))
    codes = _round_away((xg - bias[..., None]) / scale[..., None])
    codes = codes.clamp(0, (1 << bits) - 1).to(torch.int32).flatten(-2)
    return codes, scale, bias


def _pack(codes, bits):
    per = 32 // bits
    c = codes.unflatten(-1, (-1, per))
    out = c[..., 0].clone()
    for i in range(1, per):
        out |= c[..., i] << (bits * i)
    return out


def _fill_pool(pool, case, gen):
    """Quantized N(0, 1) keys (four channels of each head eight times as large)
    and values in every row of the pool."""
    kc, kp, vc, vp = _components(pool, case)
    d, hkv = case["d"], case["hkv"]
    boost = torch.ones(hkv, 1, 1, d, device=DEVICE)
    for h in range(hkv):
        ch = torch.randperm(d, generator=gen, device=DEVICE)[:4]
        boost[h, 0, 0, ch] = 8.0
    step = max(1, (1 << 26) // (hkv * case["page"] * d))
    dt = _torch_dtype(case)
    for p0 in range(0, pool.shape[0], step):
        p1 = min(pool.shape[0], p0 + step)
        shape = (p1 - p0, hkv, case["page"] // TILE, TILE, d)
        for codes, pairs, mul in ((kc, kp, boost), (vc, vp, None)):
            x = torch.randn(shape, generator=gen, device=DEVICE)
            if mul is not None:
                x *= mul
            c, s, b = _quantise(x.to(dt).float(), case["bits"], case["gs"])
            codes[p0:p1] = _pack(c, case["bits"])
            pairs[p0:p1, ..., 0] = s.to(dt)
            pairs[p0:p1, ..., 1] = b.to(dt)


def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-bun_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import kvq
    return kvq


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    lens, rows = _shape(case)
    page, hkv, hq, d = case["page"], case["hkv"], case["hq"], case["d"]
    dt = _torch_dtype(case)
    w, g = _row_words(case)
    need = [-(-n // page) for n in lens]
    # the pages of each sequence lie scattered over the pool; table entries
    # past a sequence's last page are unset
    order = torch.randperm(sum(need), generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pool = torch.empty(sum(need), hkv, page // TILE, 2 * TILE * (w + g), dtype=torch.int32,
                       device=DEVICE)
    _fill_pool(pool, case, gen)
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    st = dict(case=case, lens=lens, rows=rows, cu=cu, pool=pool, table=table,
              seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEVICE),
              cu_rows=torch.tensor(cu, dtype=torch.int32, device=DEVICE))
    total = cu[-1] + case.get("pad", 0)
    if case["op"] == "append":
        # q, k and v as a layer's fused projection leaves them
        qkv = torch.randn(total, hq + 2 * hkv, d, generator=gen, device=DEVICE).to(dt)
        st["qkv"] = qkv
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        st["q_out"] = torch.zeros(total, hq, d, dtype=dt, device=DEVICE)
        st["freqs"] = None
        if case["table"] and case["rope_dims"]:
            i = torch.arange(case["rope_dims"] // 2, dtype=torch.float64, device=DEVICE)
            st["freqs"] = (case["base"] ** (2.0 * i / case["rope_dims"])).float()
    else:
        st["q"] = torch.randn(total, hq, d, generator=gen, device=DEVICE).to(dt)
        st["out"] = torch.zeros(total, hq, d, dtype=dt, device=DEVICE)
        st["scale"] = 1.0 / math.sqrt(d)
    if own:
        kvq = _framework()
        st["cache"] = kvq.PagedQuantizedKVCache(pool.shape[0], page, hkv, d, case["gs"],
                                                case["bits"], dt, pool=pool)
        if case["op"] == "append":
            st["rope"] = kvq.Rope(case["rope_dims"], base=case["base"], freqs=st["freqs"],
                                  traditional=case["traditional"])
    return st


# --------------------------------------------------------------- one pass --

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _append_outputs(st):
    """The pool's components as they are held: the packed codes are whole
    numbers, the scales and biases are values of the dtype."""
    kc, kp, vc, vp = _components(st["pool"], st["case"])
    return {"k_codes": kc, "k_scales_biases": kp, "v_codes": vc, "v_scales_biases": vp,
            "q": st["q_out"]}


def _run_own(st):
    case, cache = st["case"], st["cache"]
    if case["op"] == "append":
        cache.append(st["k"], st["v"], st["table"], st["seq_lens"], st["cu_rows"],
                     rope=st["rope"], q=st["q"], q_out=st["q_out"])
        return _append_outputs(st)
    if case["op"] == "decode":
        return cache.sdpa_decode(st["q"], st["table"], st["seq_lens"], st["scale"],
                                 window=case["window"], sinks=case["sinks"], out=st["out"])
    return cache.sdpa_prefill(st["q"], st["table"], st["seq_lens"], st["cu_rows"], st["scale"],
                              window=case["window"], sinks=case["sinks"], out=st["out"])


def _rows_of(st, b, pos):
    """Page, tile and row of positions `pos` (a device tensor) of sequence b."""
    page = st["case"]["page"]
    return st["table"][b, pos // page].long(), (pos % page) // TILE, pos % TILE


def _rotate(x, pos, case, freqs):
    """x [n, heads, d] at positions pos: rotated in 64 bits, back in x's type."""
    dims = case["rope_dims"]
    if not dims:
        return x
    half = dims // 2
    if freqs is not None:
        inv = 1.0 / freqs.double()
    else:
        i = torch.arange(half, dtype=torch.float64, device=x.device)
        inv = torch.full_like(i, case["base"]) ** (-2.0 * i / dims)
    ang = pos.double()[:, None, None] * inv
    c, s = torch.cos(ang), torch.sin(ang)
    y = x.double()
    if case["traditional"]:
        a, b = y[..., 0:dims:2], y[..., 1:dims:2]
    else:
        a, b = y[..., :half], y[..., half:dims]
    u, v = a * c - b * s, a * s + b * c
    rot = torch.stack([u, v], -1).flatten(-2) if case["traditional"] else torch.cat([u, v], -1)
    return torch.cat([rot, y[..., dims:]], -1).float().to(x.dtype)


def _run_plain(st):
    case = st["case"]
    if case["op"] == "append":
        kc, kp, vc, vp = _components(st["pool"], case)
        dt = st["k"].dtype
        for b, (n, r) in enumerate(zip(st["lens"], st["rows"])):
            t0 = st["cu"][b]
            pos = torch.arange(n - r, n, device=DEVICE)
            pg, tile, row = _rows_of(st, b, pos)
            st["q_out"][t0:t0 + r] = _rotate(st["q"][t0:t0 + r], pos, case, st["freqs"])
            k = _rotate(st["k"][t0:t0 + r], pos, case, st["freqs"])
            for x, codes, pairs in ((k, kc, kp), (st["v"][t0:t0 + r], vc, vp)):
                c, s, z = _quantise(x.float(), case["bits"], case["gs"])
                codes[pg, :, tile, row] = _pack(c, case["bits"])
                pairs[pg, :, tile, row] = torch.stack([s, z], -1).to(dt)
        return _append_outputs(st)
    window, sinks = case["window"], case["sinks"]
    rep = case["hq"] // case["hkv"]
    for b, (n, r) in enumerate(zip(st["lens"], st["rows"])):
        t0, first = st["cu"][b], n - r
        lo = max(0, first - window + 1) if window > 0 else 0
        head = min(max(sinks, 0), lo)
        pos = torch.cat([torch.arange(head, device=DEVICE), torch.arange(lo, n, device=DEVICE)])
        k, v = _plain_rows(st, b, pos)  # [keys, heads, d] f32
        q = st["q"][t0:t0 + r].float().unflatten(1, (case["hkv"], rep))
        qpos = torch.arange(first, n, device=DEVICE)[:, None]
        see = pos[None] <= qpos
        if window > 0:
            see &= (pos[None] > qpos - window) | (pos[None] < sinks)
        for h in range(case["hkv"]):
            s = q[:, h].flatten(0, 1) @ k[:, h].T
            s = s.unflatten(0, (r, rep)) * st["scale"]
            s = s.masked_fill(~see[:, None], float("-inf"))
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = (e.flatten(0, 1) @ v[:, h]).unflatten(0, (r, rep)) / e.sum(-1, keepdim=True)
            st["out"][t0:t0 + r, h * rep:(h + 1) * rep] = o.to(st["out"].dtype)
    return st["out"]


def _plain_rows(st, b, pos):
    case = st["case"]
    kc, kp, vc, vp = _components(st["pool"], case)
    pg, tile, row = _rows_of(st, b, pos)
    shift = torch.arange(0, 32, case["bits"], device=DEVICE, dtype=torch.int32)
    out = []
    for codes, pairs in ((kc, kp), (vc, vp)):
        w = codes[pg, :, tile, row]
        c = ((w[..., None] >> shift) & ((1 << case["bits"]) - 1)).flatten(-2).float()
        p = pairs[pg, :, tile, row].float()
        x = c.unflatten(-1, (-1, case["gs"])) * p[..., 0:1] + p[..., 1:2]
        out.append(x.flatten(-2))
    return out


# --------------------------------------------- the definition in 64 bits --

def exact(case, seed):
    """What run returns, in 64 bits (the appended codes by the rule's own
    32-bit steps, which define them), written apart from the plain form."""
    lens, rows = _shape(case)
    if case["op"] == "append":
        return _exact_append(case, seed, lens, rows)
    return _exact_attention(case, seed, lens, rows)


def _np_quantise(x, bits, gs):
    f = np.float32
    g = x.astype(f).reshape(-1, gs)
    top = f((1 << bits) - 1)
    lo, hi = g.min(1), g.max(1)
    step = np.maximum((hi - lo) / top, f(QUANT_EPS))
    low_wins = np.abs(lo) > np.abs(hi)
    edge = np.where(low_wins, lo, hi)
    step = np.where(low_wins, step, -step)
    away = lambda t: np.where(np.abs(t - np.trunc(t)) >= f(0.5), np.trunc(t) + np.sign(t), np.trunc(t))
    k = away(edge / step)
    with np.errstate(divide="ignore", invalid="ignore"):
        scale = np.where(k != 0, edge / k, step).astype(f)
    bias = np.where(k != 0, edge, f(0)).astype(f)
    code = np.clip(away((g - bias[:, None]) / scale[:, None]), 0, top).astype(np.uint32)
    per = 32 // bits
    words = np.zeros((code.size // per,), np.uint32)
    flat = code.reshape(-1, per)
    for i in range(per):
        words |= flat[:, i] << np.uint32(bits * i)
    return words.view(np.int32), scale, bias


def _exact_append(case, seed, lens, rows):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    dt, d, dims, page = st["k"].dtype, case["d"], case["rope_dims"], case["page"]
    w, g = _row_words(case)
    pool = st["pool"].cpu()
    table = st["table"].cpu().numpy()
    bufs = {n: st[n].cpu() for n in ("q", "k", "v")}
    freqs = None if st["freqs"] is None else st["freqs"].cpu().numpy().astype(np.float64)
    q_out = torch.zeros(st["q_out"].shape, dtype=torch.float64)
    parts = [t.clone() for t in _components(pool, case)]
    i = np.arange(dims // 2, dtype=np.float64)
    inv = 1.0 / freqs if freqs is not None else np.power(case["base"], -2.0 * i / max(dims, 1))

    def turn(x, pos):  # numpy f64 [n, heads, d]
        y = x.copy()
        if dims:
            ang = pos[:, None].astype(np.float64) * inv[None]
            z = np.exp(1j * ang)[:, None]
            if case["traditional"]:
                r = (x[..., 0:dims:2] + 1j * x[..., 1:dims:2]) * z
                y[..., 0:dims:2], y[..., 1:dims:2] = r.real, r.imag
            else:
                r = (x[..., :dims // 2] + 1j * x[..., dims // 2:dims]) * z
                y[..., :dims // 2], y[..., dims // 2:dims] = r.real, r.imag
        return y

    to64 = lambda t: t.double().numpy()
    t0 = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        pos = np.arange(n - r, n)
        pg = torch.from_numpy(table[b][pos // page].astype(np.int64))
        tile, row = torch.from_numpy(pos % page // TILE), torch.from_numpy(pos % TILE)
        q_out[t0:t0 + r] = torch.from_numpy(turn(to64(bufs["q"][t0:t0 + r]), pos))
        k = torch.from_numpy(turn(to64(bufs["k"][t0:t0 + r]), pos)).float().to(dt).float().numpy()
        for x, codes, pairs in ((k, parts[0], parts[1]),
                                (bufs["v"][t0:t0 + r].float().numpy(), parts[2], parts[3])):
            c, s, z = _np_quantise(x, case["bits"], case["gs"])
            codes[pg, :, tile, row] = torch.from_numpy(c.reshape(r, -1, w))
            sz = torch.from_numpy(np.stack([s, z], -1).reshape(r, -1, g, 2))
            pairs[pg, :, tile, row] = sz.to(dt)
        t0 += r
    names = ("k_codes", "k_scales_biases", "v_codes", "v_scales_biases")
    out = dict(zip(names, parts))
    out["q"] = q_out
    return out


def _exact_attention(case, seed, lens, rows):
    global own
    keep, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = keep
    d, gs, bits, hkv = case["d"], case["gs"], case["bits"], case["hkv"]
    rep, page = case["hq"] // hkv, case["page"]
    w, g = _row_words(case)
    dt = st["q"].dtype
    flat = st["pool"].flatten(2)  # [pages, heads, words of a page]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=DEVICE)
    half = TILE * (w + g)
    t0 = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        pages = flat[st["table"][b, :-(-n // page)].long()]
        tiles = pages.unflatten(-1, (page // TILE, 2, half)).permute(1, 3, 0, 2, 4)
        qpos = torch.arange(n - r, n, device=DEVICE)[:, None]
        j = torch.arange(n, device=DEVICE)[None]
        bar = j > qpos
        if case["window"] > 0:
            bar |= (qpos - j >= case["window"]) & (j >= case["sinks"])
        for h in range(hkv):
            x = []
            for part in range(2):
                t = tiles[h, part].reshape(-1, half)
                c = t[:, :TILE * w].reshape(-1, w)[:n]
                z = t[:, TILE * w:].contiguous().view(dt).reshape(-1, g, 2)[:n].double()
                codes = torch.stack([(c >> s) & ((1 << bits) - 1) for s in range(0, 32, bits)], -1)
                codes = codes.reshape(n, g, gs).double()
                x.append((codes * z[..., :1] + z[..., 1:]).reshape(n, d))
            for i in range(rep):
                q = st["q"][t0:t0 + r, h * rep + i].double()
                s = (q @ x[0].T) * st["scale"]
                p = torch.softmax(s.masked_fill(bar, -math.inf), -1)
                out[t0:t0 + r, h * rep + i] = p @ x[1]
        t0 += r
    return out
