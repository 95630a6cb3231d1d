"""Plain 64-bit forms of the 8-bit KV operators and of the rotary ones, on the CPU, token by token, for the tests.

Codes follow the format's own rounding points (fp32 products and sums in the rotation), so codes, scales and rotated rows
are compared for equality; attention is compared within bounds that `attend_tolerance` derives from the inputs alone."""
import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def f32(x):
    return x.to(torch.float32).double()


def rotate(x, cos, sin, interleaved):
    """x [N, heads, hd] fp64 holding the storage values; cos / sin [N, r / 2]. Products and sums rounded to fp32."""
    r = 2 * cos.shape[1]
    out = x.clone()
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        c, s = cos[:, None, i].double(), sin[:, None, i].double()
        xa, xb = x[..., a], x[..., b]
        out[..., a] = f32(f32(xa * c) - f32(xb * s))
        out[..., b] = f32(f32(xb * c) + f32(xa * s))
    return out


def pow2_scale(amax: float, qmax: float) -> float:
    if not math.isfinite(amax):
        return float("nan")
    s = 2.0 ** -100
    while amax > qmax * s:
        s *= 2
    return s


def encode(y: torch.Tensor, dtype) -> torch.Tensor:
    """fp64 quotients -> the values of the nearest codes (ties to even); NaN -> 0."""
    y = torch.nan_to_num(y, nan=0.0, posinf=1e300, neginf=-1e300)
    if dtype == torch.int8:
        return torch.round(y).clamp(-127, 127)
    mag = y.abs().clamp(max=448.0)
    _, e = torch.frexp(mag)
    step = torch.ldexp(torch.ones_like(mag), torch.clamp(e - 1, min=-6) - 3)
    return torch.copysign(torch.round(mag / step) * step, y)


def append(pool, scale, x, slots):
    """One plane set: pool [nb, bs, nkv, hd] of codes, scale [nb, nkv], x [N, nkv, hd] fp64, slots list. Returns (codes
    as fp64 values, scales fp64)."""
    nb, bs, nkv, hd = pool.shape
    codes, sc = pool.float().double().clone(), scale.double().clone()
    rows = {}
    for t, s in enumerate(slots):
        if 0 <= s < nb * bs:
            rows.setdefault(s // bs, {})[s % bs] = t
    for b, where in rows.items():
        for h in range(nkv):
            vals = torch.stack([x[t, h] for t in where.values()])
            amax = float("nan") if bool(vals.isnan().any()) else vals.abs().max().item()
            s = pow2_scale(amax, QMAX[pool.dtype])
            if 0 in where:
                codes[b, :, h] = 0.0
            else:
                old = sc[b, h].item()
                s = float("nan") if (math.isnan(s) or math.isnan(old)) else max(s, old)
                if s != old:
                    ratio = f32(torch.tensor(old / s if s == s else float("nan"), dtype=torch.float64))
                    codes[b, :, h] = encode(f32(codes[b, :, h] * ratio), pool.dtype)
            inv = f32(torch.tensor(1.0 / s, dtype=torch.float64))
            for off, t in where.items():
                codes[b, off, h] = encode(f32(x[t, h] * inv), pool.dtype)
            sc[b, h] = s
    return codes, sc


def values(pool, scale):
    return pool.float().double() * scale.double()[:, None, :, None]


def attend(q, kv, vv, tables, seq_lens, cu, scale, block_size, n_blocks=None, table_rows=None, fill=0.0):
    """q [N, NH, HD]; kv / vv fp64 values of the pools [nb, bs, nkv, hd]. Rows of no sequence keep `fill`."""
    N, NH, HD = q.shape
    nb, bs, nkv, _ = kv.shape
    n_blocks = nb if n_blocks is None else n_blocks
    out = torch.full((N, NH, HD), float(fill), dtype=torch.float64)
    lens = seq_lens.tolist()
    cu = list(range(len(lens) + 1)) if cu is None else cu.tolist()
    for s, L in enumerate(lens):
        T = cu[s + 1] - cu[s]
        row = tables[s if table_rows is None else int(table_rows[s])].tolist()
        L = max(0, min(L, len(row) * bs))
        keys = [(row[t // bs], t % bs, t) for t in range(L) if 0 <= row[t // bs] < n_blocks]
        for j in range(T):
            see = [(b, o) for b, o, t in keys if t <= L - T + j]
            for h in range(NH):
                g = h // (NH // nkv)
                if not see:
                    out[cu[s] + j, h] = 0.0
                    continue
                bi, oi = torch.tensor([x[0] for x in see]), torch.tensor([x[1] for x in see])
                sc = (kv[bi, oi, g] @ q[cu[s] + j, h].double()) * scale
                out[cu[s] + j, h] = torch.softmax(sc, 0) @ vv[bi, oi, g]
    return out


def attend_fast(q, kv, vv, tables, seq_lens, cu, scale):
    """The same for plain batches (every block id valid), one product per sequence and KV head."""
    N, NH, HD = q.shape
    nb, bs, nkv, _ = kv.shape
    out = torch.zeros(N, NH, HD, dtype=torch.float64)
    lens = seq_lens.tolist()
    cu = list(range(len(lens) + 1)) if cu is None else cu.tolist()
    grp = NH // nkv
    for s, L in enumerate(lens):
        a, T = cu[s], cu[s + 1] - cu[s]
        if T == 0:
            continue
        if L <= 0:
            continue
        ids = tables[s, :-(-L // bs)].long()
        k, v = kv[ids].reshape(-1, nkv, HD)[:L], vv[ids].reshape(-1, nkv, HD)[:L]
        vis = torch.arange(L)[None] <= (L - T + torch.arange(T))[:, None]
        for h in range(NH):
            sc = (q[a:a + T, h].double() @ k[:, h // grp].t()) * scale
            p = torch.softmax(sc.masked_fill(~vis, float("-inf")), 1)
            out[a:a + T, h] = torch.nan_to_num(p @ v[:, h // grp])
    return out


def attend_tolerance(q, kv, vv, tables, seq_lens, scale, ref, out_dtype, p_bits):
    """Bound on |kernel - exact|, from the inputs:
      scores: a dot of HD products accumulated in fp32 is off by at most (HD + 4) 2^-23 sum|q k| (2^-23, not 2^-24: the tensor
      cores may truncate), and as much again for the factors applied to it; exp turns that into the same relative error of
      a weight, exp2's own is 2^-22; numerator and denominator each carry it, so 2x.
      weights: rounded to p_bits bits before they meet V (p_bits = None: not rounded), relative 2^-p_bits half steps, counted whole.
      sums over L keys in fp32: (L + 8) 2^-23.
      All of it scales the largest |v|; the output rounds by eps / 2 of its own dtype."""
    HD = q.shape[-1]
    lens = seq_lens.clamp(min=1)
    dot = q.double().abs().amax() * kv.abs().amax() * HD * scale        # a generous sum|q k| scale
    rel = 2 * (2 * (HD + 4) * 2.0 ** -23 * float(dot) + 2.0 ** -22) + 2 * (float(lens.max()) + 8) * 2.0 ** -23
    if p_bits is not None:
        rel += 2.0 ** -p_bits
    return rel * float(vv.abs().amax()) + torch.finfo(out_dtype).eps / 2 * ref.abs()
