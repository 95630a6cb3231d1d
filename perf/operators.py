"""Operator workloads: rotary position tables, the rotation + cache append, and attention over the paged KV cache, for
16/32-bit and 8-bit pools.

`run` computes an operator either in its plain form (elementary torch operations in 32 bits, 64 where angles need it) or,
with `own` set, through this package's entry points. Sizes are those of the benchmark configurations and of the layer
shapes in nanoserve_b200/synthetic.py; every length is drawn from the case itself, every value from the seed.

Definitions shared by all forms (the rounding points are part of them):
  tables   cos/sin[t, i] = factor * cos/sin(position_t * f_i), rounded once to fp32
  rotate   pair (a, b) -> (a c - b s, b c + a s) in fp32, each product and each sum rounded, then once to the output type;
           pairs are (i, i + r/2) in the half layout, (2i, 2i + 1) in the interleaved one, dims past r are copied
  append   16/32-bit pools: row slot of the pool = the token's rotated key / its value; a slot outside the pool stores
           nothing.
           8-bit pools hold codes and one scale per block and KV head (K and V apart). The rows of a block that a call
           writes have a largest magnitude A; S = the smallest power of two >= 2^-100 with A <= Q S (Q = 127 for int8,
           448 for e4m3). A call that writes a block's first row starts the block afresh: scale = S, rows it does not
           write hold code 0. Otherwise the scale becomes max(scale, S) and the other rows' codes are rounded again to it.
  attend   softmax over the visible keys of scale * q.k, times v, keys and values = code * their block's scale
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_KV = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
_QMAX = {"int8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------------------------------------------ cases
def listed():
    half = {"layout": "half", "dtype": "bf16"}
    inter = {"layout": "interleaved", "dtype": "bf16"}
    return [
        # the tables of a 64-row decode step whose rows sit far out in a long context, and of a large prefill step
        {"name": "tables-decode64-far", "op": "tables", "tokens": 64, "rot": 64, "far": 1000000, "shape_seed": 1},
        {"name": "tables-8192", "op": "tables", "tokens": 8192, "rot": 128, "far": 131072, "shape_seed": 2},
        # one layer's rotation + KV store into a 16-bit pool: 32 decode rows with half of each head rotated in
        # neighbouring pairs, and a prefill step of the 28-head layer shape
        {"name": "append16-decode32-interleaved", "op": "append", "kv": "bf16", "nh": 14, "nkv": 2, "hd": 64, "rot": 32, **inter,
         "rows": 32, "lo": 64, "hi": 4096, "chunks": 0, "chunk": 0, "pad": 0, "shape_seed": 3},
        {"name": "append16-prefill-4x1024", "op": "append", "kv": "bf16", "nh": 28, "nkv": 4, "hd": 128, "rot": 128, **half,
         "rows": 0, "lo": 1, "hi": 1, "chunks": 4, "chunk": 1024, "pad": 0, "shape_seed": 4},
        # the same into an 8-bit pool: a decode step padded to its graph bucket (every row re-opens a part-filled block), and
        # a mixed step of 37 decode rows beside four chunks that start in the middle of a block
        {"name": "append8-decode61-pad3", "op": "append", "kv": "int8", "nh": 14, "nkv": 2, "hd": 64, "rot": 64, **half,
         "rows": 61, "lo": 64, "hi": 4096, "chunks": 0, "chunk": 0, "pad": 3, "shape_seed": 5},
        {"name": "append8-mixed-37+4x1021", "op": "append", "kv": "e4m3", "nh": 28, "nkv": 4, "hd": 128, "rot": 128, **half,
         "rows": 37, "lo": 64, "hi": 4096, "chunks": 4, "chunk": 1021, "pad": 0, "shape_seed": 6},
        # decode attention: one short request alone (latency), the benchmark's 48 ragged rows, 64 rows of the 28-head
        # shape, and two requests at a 128K context
        {"name": "attend-decode1-short", "op": "attend", "kv": "int8", "nh": 14, "nkv": 2, "hd": 64, "dtype": "bf16",
         "rows": 1, "lo": 300, "hi": 300, "chunks": 0, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0, "shape_seed": 7},
        {"name": "attend-decode48-ragged", "op": "attend", "kv": "int8", "nh": 14, "nkv": 2, "hd": 64, "dtype": "bf16",
         "rows": 48, "lo": 128, "hi": 8192, "chunks": 0, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0, "shape_seed": 8},
        {"name": "attend-decode64-28heads", "op": "attend", "kv": "e4m3", "nh": 28, "nkv": 4, "hd": 128, "dtype": "bf16",
         "rows": 64, "lo": 256, "hi": 4608, "chunks": 0, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0, "shape_seed": 9},
        {"name": "attend-decode2-128k", "op": "attend", "kv": "int8", "nh": 12, "nkv": 2, "hd": 128, "dtype": "bf16",
         "rows": 2, "lo": 130001, "hi": 131072, "chunks": 0, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0, "shape_seed": 10},
        # mixed step of the benchmark (48 decode rows + four 512-token chunks) and one long chunk on a long cached prompt
        {"name": "attend-mixed-48+4x512", "op": "attend", "kv": "int8", "nh": 14, "nkv": 2, "hd": 64, "dtype": "bf16",
         "rows": 48, "lo": 128, "hi": 8192, "chunks": 4, "chunk": 512, "ctx_lo": 0, "ctx_hi": 2048, "shape_seed": 11},
        {"name": "attend-prefill-2048-on-6k", "op": "attend", "kv": "e4m3", "nh": 28, "nkv": 4, "hd": 128, "dtype": "bf16",
         "rows": 0, "lo": 1, "hi": 1, "chunks": 1, "chunk": 2048, "ctx_lo": 6001, "ctx_hi": 6001, "shape_seed": 12},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


_HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (14, 2, 128), (7, 1, 128), (16, 2, 128)]


def draw(rng: random.Random):
    """One more case of the same ranges."""
    op = rng.choice(["tables", "append", "append", "attend", "attend", "attend"])
    seed = rng.randrange(1 << 30)
    if op == "tables":
        return {"op": op, "tokens": _log(rng, 1, 8192), "rot": 2 * _log(rng, 8, 64), "far": _log(rng, 4096, 1000000), "shape_seed": seed}
    nh, nkv, hd = rng.choice(_HEADS)
    if op == "append":
        kv = rng.choice(["int8", "e4m3", "bf16", "fp32"])
        case = {"op": op, "kv": kv, "nh": nh, "nkv": nkv, "hd": hd, "rot": rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)]),
                "layout": rng.choice(["half", "interleaved"]),
                "dtype": kv if kv in _DTYPES else rng.choice(["bf16", "bf16", "fp32"]),
                "rows": _log(rng, 1, 96), "lo": 1, "hi": 4096, "chunks": rng.choice([0, 0, 1, 3]), "chunk": _log(rng, 2, 640),
                "pad": rng.choice([0, 0, 3]), "shape_seed": seed}
        return case
    hi = _log(rng, 1, 16384)
    rows = _log(rng, 1, max(1, min(96, 200000 // hi)))
    case = {"op": op, "kv": rng.choice(["int8", "e4m3"]), "nh": nh, "nkv": nkv, "hd": hd, "dtype": rng.choice(["bf16", "bf16", "bf16", "fp32"]),
            "rows": rows, "lo": max(1, hi // rng.choice([1, 2, 64])), "hi": hi, "chunks": 0, "chunk": 0, "ctx_lo": 0, "ctx_hi": 0,
            "shape_seed": seed}
    if case["dtype"] == "bf16" and rng.random() < 0.45:
        case.update(chunks=rng.randint(1, 4), chunk=_log(rng, 2, 640), ctx_lo=0, ctx_hi=_log(rng, 1, 4096))
        if rng.random() < 0.3:
            case["rows"] = 0
    return case


def _lengths(case):
    """(context before the step, new tokens) of every sequence; decode rows first."""
    r = random.Random(case["shape_seed"])
    out = [(r.randint(case["lo"], case["hi"]) - 1, 1) for _ in range(case["rows"])]
    if case["op"] == "attend":
        return out + [(r.randint(case["ctx_lo"], case["ctx_hi"]), case["chunk"]) for _ in range(case["chunks"])]
    return out + [(r.randint(0, 2000) if i % 2 else 0, case["chunk"]) for i in range(case["chunks"])]


# ------------------------------------------------------------------------------------------------------ inputs
def _pow2_scale(amax, qmax):
    """Smallest power of two s >= 2^-100 with amax <= qmax * s; NaN where amax is not finite."""
    m, e = torch.frexp(amax)
    qm, qe = math.frexp(qmax)
    s = torch.ldexp(torch.ones_like(amax), e - qe + (m > qm).to(e.dtype)).clamp(min=2.0 ** -100)
    s = torch.where(amax == 0, torch.full_like(s, 2.0 ** -100), s)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


def _to_codes(x, kv):
    """Values already divided by their scale -> codes (ties to even)."""
    if kv == "int8":
        return torch.nan_to_num(x).round().clamp(-127, 127).to(torch.int8)
    return torch.nan_to_num(x).clamp(-448, 448).to(torch.float8_e4m3fn)


def _random_pool(g, kv, blocks, nkv, hd):
    """Codes and scales as appends leave them: N(0, 1) values whose size differs from head to head."""
    dev = "cuda"
    pool = torch.empty(blocks, BLOCK, nkv, hd, dtype=_KV[kv], device=dev)
    scale = torch.empty(blocks, nkv, dtype=torch.float32, device=dev)
    size = torch.rand(nkv, 1, generator=g, device=dev) * 2 + 0.25
    step = max(1, (1 << 26) // (BLOCK * nkv * hd))
    for a in range(0, blocks, step):
        x = torch.randn(min(step, blocks - a), BLOCK, nkv, hd, generator=g, device=dev) * size
        s = _pow2_scale(x.abs().amax(dim=(1, 3)), _QMAX[kv])
        pool[a:a + step] = _to_codes(x / s[:, None, :, None], kv)
        scale[a:a + step] = s
    return pool, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + case["shape_seed"])
    dev = "cuda"
    op = case["op"]
    if op == "tables":
        n, half = case["tokens"], case["rot"] // 2
        pos = torch.randint(0, case["far"], (n,), generator=g, device=dev, dtype=torch.int64)
        inv = (1e6 ** (-torch.arange(half, dtype=torch.float64) / half)).float().to(dev)
        return {"op": op, "positions": pos, "inv_freq": inv, "factor": 1.0 + 0.1 * math.log(4.0)}
    seqs = _lengths(case)
    nh, nkv, hd, dtype = case["nh"], case["nkv"], case["hd"], _DTYPES[case["dtype"]]
    if op == "append":
        n_tok = sum(t for _, t in seqs)
        N = n_tok + case["pad"]
        need = [(c + t - 1) // BLOCK - c // BLOCK + 1 for c, t in seqs]         # blocks of the sequence that the call touches
        blocks = sum(need) + 8
        perm = torch.randperm(blocks, generator=g, device=dev)
        slots, used = [], 0
        for (c, t), nb in zip(seqs, need):
            p = torch.arange(c % BLOCK, c % BLOCK + t, device=dev)
            slots.append(perm[used:used + nb][p // BLOCK] * BLOCK + p % BLOCK)
            used += nb
        slots.append(torch.full((case["pad"],), -1, dtype=torch.int64, device=dev))
        half = case["rot"] // 2
        pos = torch.cat([torch.arange(c, c + t) for c, t in seqs] + [torch.zeros(case["pad"])]).double()
        ang = pos[:, None] * 1e6 ** (-torch.arange(half, dtype=torch.float64) / half)
        st = {"op": op, "case": case, "slots": torch.cat(slots).to(torch.int64),
              "qkv": (torch.randn(N, (nh + 2 * nkv) * hd, generator=g, device=dev) * 1.5).to(dtype),
              "cos": ang.cos().float().to(dev), "sin": ang.sin().float().to(dev)}
        if case["kv"] in _KV:
            st["k"], st["k_scale"] = _random_pool(g, case["kv"], blocks, nkv, hd)
            st["v"], st["v_scale"] = _random_pool(g, case["kv"], blocks, nkv, hd)
        else:
            st["k"] = torch.randn(blocks, BLOCK, nkv, hd, generator=g, device=dev).to(dtype)
            st["v"] = torch.randn(blocks, BLOCK, nkv, hd, generator=g, device=dev).to(dtype)
        return st
    lens = [c + t for c, t in seqs]
    news = [t for _, t in seqs]
    need = [-(-L // BLOCK) for L in lens]
    blocks = sum(need) + 8
    perm = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    tables = torch.zeros(len(seqs), max(need), dtype=torch.int32, device=dev)
    used = 0
    for i, nb in enumerate(need):
        tables[i, :nb] = perm[used:used + nb]
        used += nb
    N = sum(news)
    st = {"op": op, "case": case, "lens": lens, "news": news, "tables": tables, "scale": hd ** -0.5,
          "q": (torch.randn(N, nh, hd, generator=g, device=dev) * 1.5).to(dtype),
          "seq_lens": torch.tensor(lens, dtype=torch.int32, device=dev),
          "cu": torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device=dev)}
    st["k"], st["k_scale"] = _random_pool(g, case["kv"], blocks, nkv, hd)
    st["v"], st["v_scale"] = _random_pool(g, case["kv"], blocks, nkv, hd)
    if own:
        # a serving step plans once and attends in every layer: the workspace and its plan exist before the call
        from nanoserve_b200.kernels.paged_attention import AttnWorkspace
        st["workspace"] = AttnWorkspace(max(len(seqs), 1), max(N, 1), nh, hd)
        if case["chunks"]:
            st["workspace"].plan(st["seq_lens"], st["cu"], len(seqs), BLOCK)
    return st


# ------------------------------------------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, layout):
    """x fp32 [N, heads, hd]; cos / sin [N, r/2]."""
    half = cos.shape[1]
    c, s = cos[:, None, :], sin[:, None, :]
    out = x.clone()
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return out


def _last_writer(slots, n_slots):
    """[n_slots + 1] index of the last token that names each slot, -1 where none does (the last entry takes the strays)."""
    n = slots.shape[0]
    where = torch.where((slots >= 0) & (slots < n_slots), slots, torch.full_like(slots, n_slots))
    idx = torch.full((n_slots + 1,), -1, dtype=torch.int64, device=slots.device)
    return idx.scatter_reduce_(0, where, torch.arange(n, device=slots.device), "amax")


def _append8_plain(pool, scale, x, slots, kv):
    nb, bs, nkv, hd = pool.shape
    idx = _last_writer(slots, nb * bs)[:-1].view(nb, bs)
    wrote = idx >= 0
    vals = x[idx.clamp(min=0)]                                                    # [nb, bs, nkv, hd]
    amax = torch.where(wrote[:, :, None, None], vals.abs(), torch.zeros_like(vals)).amax(dim=(1, 3))
    s = _pow2_scale(amax, _QMAX[kv])
    fresh, touched = wrote[:, :1], wrote.any(dim=1, keepdim=True)
    new = torch.where(touched, torch.where(fresh, s, torch.maximum(scale, s)), scale)
    ratio = torch.where(new == scale, torch.ones_like(new), scale / new)
    kept = _to_codes(pool.float() * ratio[:, None, :, None], kv).float()
    kept = torch.where(fresh[:, :, None, None], torch.zeros_like(kept), kept)
    code = _to_codes(vals * (1.0 / new)[:, None, :, None], kv).float()
    code = torch.where(wrote[:, :, None, None], code, torch.where(touched[:, :, None, None], kept, pool.float()))
    pool.copy_(code.to(pool.dtype))
    scale.copy_(new)


def _values(pool, scale):
    return pool.float() * scale[:, None, :, None]


def _run_append(st):
    case = st["case"]
    nh, nkv, hd, kv = case["nh"], case["nkv"], case["hd"], case["kv"]
    if own:
        from nanoserve_b200.kernels.rotary import kv_values, rope_append
        q, _, _ = rope_append(st["qkv"], st["cos"], st["sin"], nh, nkv, hd, st["k"], st["v"], st["slots"],
                              k_scale=st.get("k_scale"), v_scale=st.get("v_scale"), interleaved=case["layout"] == "interleaved")
        if kv in _KV:
            return {"q": q, "k": kv_values(st["k"], st["k_scale"]), "v": kv_values(st["v"], st["v_scale"]),
                    "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
        return {"q": q, "k": st["k"], "v": st["v"]}
    N = st["qkv"].shape[0]
    x = st["qkv"].float().view(N, nh + 2 * nkv, hd)
    qk = _rotate(x[:, :nh + nkv], st["cos"], st["sin"], case["layout"])
    q, k, v = qk[:, :nh].to(st["qkv"].dtype), qk[:, nh:], x[:, nh + nkv:]
    if kv in _KV:
        _append8_plain(st["k"], st["k_scale"], k, st["slots"], kv)
        _append8_plain(st["v"], st["v_scale"], v, st["slots"], kv)
        return {"q": q, "k": _values(st["k"], st["k_scale"]), "v": _values(st["v"], st["v_scale"]),
                "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    keep = (st["slots"] >= 0).nonzero()[:, 0] if case["pad"] else slice(None)
    st["k"].view(-1, nkv, hd)[st["slots"][keep]] = k[keep].to(st["k"].dtype)
    st["v"].view(-1, nkv, hd)[st["slots"][keep]] = v[keep].to(st["v"].dtype)
    return {"q": q, "k": st["k"], "v": st["v"]}


def _attend_plain(st):
    q, scale = st["q"], st["scale"]
    N, nh, hd = q.shape
    nkv = st["k"].shape[2]
    grp = nh // nkv
    out = torch.empty_like(q)
    a = 0
    for i, (L, T) in enumerate(zip(st["lens"], st["news"])):
        ids = st["tables"][i, :-(-L // BLOCK)].long()
        k = (st["k"][ids].float() * st["k_scale"][ids][:, None, :, None]).reshape(-1, nkv, hd)[:L]
        v = (st["v"][ids].float() * st["v_scale"][ids][:, None, :, None]).reshape(-1, nkv, hd)[:L]
        qs = q[a:a + T].float().view(T, nkv, grp, hd)
        for h in range(nkv):
            s = torch.matmul(qs[:, h].reshape(T * grp, hd), k[:, h].t()) * scale
            if T > 1:
                vis = torch.arange(L, device=q.device)[None, :] <= (L - T + torch.arange(T, device=q.device))[:, None]
                s = torch.where(vis.repeat_interleave(grp, dim=0), s, torch.full_like(s, float("-inf")))
            p = torch.exp(s - s.amax(dim=-1, keepdim=True))
            o = torch.matmul(p, v[:, h]) / p.sum(dim=-1, keepdim=True)
            out[a:a + T, h * grp:(h + 1) * grp] = o.view(T, grp, hd).to(q.dtype)
        a += T
    return out


def run(state):
    op = state["op"]
    if op == "tables":
        if own:
            from nanoserve_b200.kernels.rotary import rope_tables
            return rope_tables(state["positions"], state["inv_freq"], state["factor"])
        ang = state["positions"].double()[:, None] * state["inv_freq"].double()
        return (torch.cos(ang) * state["factor"]).float(), (torch.sin(ang) * state["factor"]).float()
    if op == "append":
        return _run_append(state)
    if own:
        from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
        cu = state["cu"] if state["case"]["chunks"] else None
        return ragged_paged_attention(state["q"], state["k"], state["v"], state["tables"], state["seq_lens"], cu, state["scale"],
                                      workspace=state["workspace"], planned=True, k_scale=state["k_scale"], v_scale=state["v_scale"])
    return _attend_plain(state)


# ------------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "tables":
        n, half = case["tokens"], case["rot"] // 2
        return {"bytes": 8 * n + 4 * half + 8 * n * half, "flops": 24.0 * n * half}
    seqs = _lengths(case)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    e = 4 if case["dtype"] == "fp32" else 2
    if op == "append":
        n_tok = sum(t for _, t in seqs)
        N = n_tok + case["pad"]
        kv8 = case["kv"] in _KV
        touched = sum((c + t - 1) // BLOCK - c // BLOCK + 1 for c, t in seqs)
        b = N * (nh + 2 * nkv) * hd * e + N * 8 + 4 * N * case["rot"] + N * nh * hd * e + n_tok * 2 * nkv * hd * (1 if kv8 else e)
        if kv8:                                  # scales of the touched blocks, then the pools read once and given out as values
            blocks = touched + 8
            b += 2 * 2 * touched * nkv * 4 + 2 * blocks * BLOCK * nkv * hd * 5 + 2 * blocks * nkv * 4
        return {"bytes": b, "flops": 3.0 * N * (nh + nkv) * case["rot"] + 2.0 * n_tok * 2 * nkv * hd * kv8}
    total = sum(c + t for c, t in seqs)
    seen = sum(t * c + t * (t + 1) // 2 for c, t in seqs)
    N = sum(t for _, t in seqs)
    nb = sum(-(-(c + t) // BLOCK) for c, t in seqs)
    return {"bytes": total * 2 * nkv * hd + nb * (2 * nkv * 4 + 4) + 2 * N * nh * hd * e + 8 * len(seqs), "flops": 4.0 * nh * hd * seen}


# ------------------------------------------------------------------------------------------------------ 64 bits
def _f32(x):
    return x.float().double()


def _exact_codes(y, kv):
    """Nearest code to y (fp64), ties to the even code, from the code tables themselves."""
    if kv == "int8":
        return torch.clamp(torch.round(y), -127, 127)
    mag = y.abs().clamp(max=448.0)
    _, e = torch.frexp(mag)
    step = torch.ldexp(torch.ones_like(mag), torch.clamp(e - 1, min=-6) - 3)
    return torch.copysign(torch.round(mag / step) * step, y)


def _exact_append8(codes, scale, x, slots, kv):
    nb, bs, nkv, hd = codes.shape
    cur, sc = codes.double().cpu(), scale.double().cpu()
    x, n_slots = x.cpu(), nb * bs
    by_block = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < n_slots:
            by_block.setdefault(s // bs, {})[s % bs] = t
    qm = _QMAX[kv]
    for b, rows in by_block.items():
        offs, toks = torch.tensor(list(rows.keys())), torch.tensor(list(rows.values()))
        xs = x[toks]                                                              # [w, nkv, hd]
        top = xs.abs().amax(dim=(0, 2))
        s = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.ceil(torch.log2((top / qm).clamp(min=2.0 ** -100))))
        s = torch.where(top > qm * s, s * 2, torch.where(top <= qm * s / 2, s / 2, s)).clamp(min=2.0 ** -100)
        if 0 in rows:
            cur[b] = 0
        else:
            s = torch.maximum(sc[b], s)
            cur[b] = _exact_codes(cur[b] * (sc[b] / s)[None, :, None], kv)
        cur[b, offs] = _exact_codes(xs / s[None, :, None], kv)
        sc[b] = s
    return (cur * sc[:, None, :, None]).to(codes.device), sc.to(codes.device)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "tables":
        turns = np.asarray(st["positions"].cpu(), dtype=np.float64)[:, None] * np.asarray(st["inv_freq"].cpu(), dtype=np.float64)
        z = np.exp(1j * turns) * st["factor"]
        return torch.from_numpy(np.ascontiguousarray(z.real)), torch.from_numpy(np.ascontiguousarray(z.imag))
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["op"] == "append":
        N, half = st["qkv"].shape[0], case["rot"] // 2
        x = st["qkv"].double().view(N, nh + 2 * nkv, hd)
        first = torch.arange(half, device=x.device) * (2 if case["layout"] == "interleaved" else 1)
        second = first + (1 if case["layout"] == "interleaved" else half)
        c, s = st["cos"].double()[:, None], st["sin"].double()[:, None]
        head = x[:, :nh + nkv]
        a, b = head[..., first], head[..., second]
        rot = head.clone()
        rot[..., first] = _f32(_f32(a * c) - _f32(b * s))                          # the definition's own rounding points
        rot[..., second] = _f32(_f32(b * c) + _f32(a * s))
        q, k, v = rot[:, :nh], rot[:, nh:], x[:, nh + nkv:]
        if case["kv"] in _KV:
            if len(st["slots"]) > 200000:
                return None
            kc, ks = _exact_append8(st["k"].float(), st["k_scale"], k, st["slots"], case["kv"])
            vc, vs = _exact_append8(st["v"].float(), st["v_scale"], v, st["slots"], case["kv"])
            return {"q": q, "k": kc, "v": vc, "k_scale": ks, "v_scale": vs}
        kp, vp = st["k"].double().view(-1, nkv, hd), st["v"].double().view(-1, nkv, hd)
        for t, slot in enumerate(st["slots"].tolist()):
            if slot >= 0:
                kp[slot], vp[slot] = k[t], v[t]
        return {"q": q, "k": kp.view(st["k"].shape), "v": vp.view(st["v"].shape)}
    grp = nh // nkv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for i, (L, T) in enumerate(zip(st["lens"], st["news"])):
        at = torch.arange(L, device="cuda")
        blk = st["tables"][i].long()[at // BLOCK]
        for h in range(nkv):
            k = st["k"][blk, at % BLOCK, h].double() * st["k_scale"][blk, h].double()[:, None]
            v = st["v"][blk, at % BLOCK, h].double() * st["v_scale"][blk, h].double()[:, None]
            for m in range(grp):
                s = torch.einsum("td,ld->tl", st["q"][row:row + T, h * grp + m].double(), k) * st["scale"]
                s.masked_fill_(at[None, :] > (L - T + torch.arange(T, device="cuda"))[:, None], float("-inf"))
                w = torch.exp(s - torch.logsumexp(s, dim=1, keepdim=True))
                out[row:row + T, h * grp + m] = torch.einsum("tl,ld->td", w, v)
        row += T
    return out
