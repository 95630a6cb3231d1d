"""Rotary positions in fp32 and the append of a step's keys and values to a paged pool, 16/32-bit or 8-bit.

`rotary_frequencies` + `rope_tables` stand beside kernels.fused.rope_cos_sin (whose tables are rounded to the model's dtype):
scaled frequencies for long contexts, angles exact for far positions, any rotary width. `rope_append` stands beside
kernels.fused.rope_qkv: either pair layout, part of the head, and pools held in 8 bits. `kv_values` reads an 8-bit pool back.
"""
from __future__ import annotations

import math

import torch

from nanoserve_b200 import _lib

KV8_DTYPES = (torch.int8, torch.float8_e4m3fn)


def rotary_frequencies(rotary_dim: int, theta: float, scaling: dict | None = None) -> tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rotary_dim / 2] on the CPU, table factor) of a model's rotary positions.

    f_i = theta^(-2 i / rotary_dim), computed in fp64 and rounded once. `scaling` is a checkpoint's rope_scaling entry; "type" (or
    "rope_type") selects
      "default"  nothing
      "linear"   f_i / factor
      "ntk"      theta * factor^(d / (d - 2)) in place of theta: the lowest frequency is divided by factor, the highest kept
      "yarn"     f_i / factor for pairs that turn less than beta_slow (1) times over original_max_position_embeddings, f_i
                 for those that turn more than beta_fast (32) times, a linear ramp over the pair index between; the tables
                 are multiplied by attention_factor (0.1 ln(factor) + 1)."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} must be positive and even")
    if not theta > 1.0:
        raise ValueError(f"rope theta {theta} must be greater than 1")
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    freq = theta ** (-i / half)
    kind = "default" if not scaling else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return freq.float(), 1.0
    factor = float(scaling.get("factor", 1.0))
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"rope scaling factor {factor} must be at least 1")
    if kind == "linear":
        return (freq / factor).float(), 1.0
    if kind == "ntk":
        if half < 2:
            raise ValueError("ntk scaling needs a rotary dim of at least 4")
        return ((theta * factor ** (rotary_dim / (rotary_dim - 2))) ** (-i / half)).float(), 1.0
    if kind == "yarn":
        span = scaling.get("original_max_position_embeddings")
        if not span:
            raise ValueError("yarn scaling needs original_max_position_embeddings")
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        # pair index at which a pair turns n times over the original context: span * theta^(-i / half) = 2 pi n
        def index(turns):
            return half * math.log(float(span) / (2.0 * math.pi * turns)) / math.log(theta)
        lo, hi = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)             # 0: keep, 1: interpolate
        att = scaling.get("attention_factor")
        att = 0.1 * math.log(factor) + 1.0 if att is None else float(att)
        return (freq * (1.0 - ramp) + freq / factor * ramp).float(), att
    raise NotImplementedError(f"rope scaling type {kind!r} (default, linear, ntk and yarn are supported)")


def rope_tables(positions: torch.Tensor, inv_freq: torch.Tensor, factor: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """factor * cos / sin of positions[t] * inv_freq[i], fp32 [T, len(inv_freq)] each (angles in fp64, rounded once)."""
    dev = _lib.same_device(positions, inv_freq)
    assert positions.dtype is torch.int64 and positions.dim() == 1 and positions.is_contiguous()
    assert inv_freq.dtype is torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous()
    t, half = positions.shape[0], inv_freq.shape[0]
    cos = inv_freq.new_empty(t, half)
    sin = torch.empty_like(cos)
    _lib.rope_tables(dev, positions.data_ptr(), inv_freq.data_ptr(), factor, cos.data_ptr(), sin.data_ptr(), t, half)
    return cos, sin


def check_kv8_scales(pool: torch.Tensor, scale: torch.Tensor | None, other: torch.Tensor | None = None) -> tuple[int, int]:
    """An 8-bit pool's scales: fp32 [num_blocks, n_kv_heads], one for K and one for V, of equal strides; returns the strides."""
    if scale is None:
        raise ValueError(f"a {pool.dtype} pool needs k_scale and v_scale (fp32 [num_blocks, n_kv_heads])")
    (blocks, _, heads, _), strides = pool.shape, scale.stride()
    shape = (blocks, heads)
    assert scale.dtype is torch.float32 and scale.shape == shape, "scales are fp32 [num_blocks, n_kv_heads]"
    if other is not None:
        assert other.dtype is torch.float32 and other.shape == shape, "scales are fp32 [num_blocks, n_kv_heads]"
        assert other.stride() == strides, "k_scale and v_scale must have equal strides"
    return strides


_NO_POOL = (0, 0, 0, 0, 0)


def _pool_args(dtype, n, n_kv_heads, head_dim, k_cache, v_cache, slots, k_scale, v_scale):
    """Checked cache layer of an append: (pointers, sizes and strides, pool dtype code)."""
    if k_cache is None:
        return _NO_POOL, 0, 1, (0, 0, 0, 0, 0), _lib.dtype_code(dtype)
    if v_cache is None or slots is None:
        raise ValueError("a cache layer needs k_cache, v_cache and slots")
    shape, strides, kv_dtype = k_cache.shape, k_cache.stride(), k_cache.dtype
    assert len(shape) == 4, "cache layer shape"
    blocks, block_size, heads, hd = shape
    assert heads == n_kv_heads and hd == head_dim and v_cache.shape == shape, "cache layer shape"
    s0, s1, s2, s3 = strides
    assert v_cache.stride() == strides and s3 == 1 and v_cache.dtype is kv_dtype
    assert slots.dtype is torch.int64 and slots.is_contiguous() and slots.shape[0] >= n
    code, sc0, sc1 = _lib.kv8_code(kv_dtype), 0, 0
    if code is None:
        assert kv_dtype is dtype, "the pool holds the activations' dtype, int8 or float8_e4m3fn"
        assert k_scale is None and v_scale is None, "scales belong to 8-bit pools"
        code = _lib.dtype_code(dtype)
        ks = vs = 0
    else:
        if v_scale is None:
            raise ValueError(f"a {kv_dtype} pool needs k_scale and v_scale (fp32 [num_blocks, n_kv_heads])")
        sc0, sc1 = check_kv8_scales(k_cache, k_scale, v_scale)
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    return (k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, slots.data_ptr()), blocks * block_size, block_size, (s0, s1, s2, sc0, sc1), code


def rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, n_heads: int, n_kv_heads: int, head_dim: int,
                k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None, slots: torch.Tensor | None = None, *,
                k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, interleaved: bool = False,
                dense_kv: bool = False):
    """qkv [N, (n_heads + 2 n_kv_heads) head_dim] (rows may be strided); cos / sin fp32 [N, r / 2] from rope_tables: the first
    r dims of every query and key head are rotated, in pairs (i, i + r/2) or, interleaved, (2i, 2i + 1). Returns
    (q, k, v): q [N, n_heads, hd]; k and v dense as well with dense_kv, else None. With a cache layer
    (k_cache / v_cache [blocks, block_size, n_kv_heads, hd], int64 slots [N]) K and V are stored there; a negative slot stores
    nothing. An int8 or float8_e4m3fn layer needs k_scale / v_scale fp32 [blocks, n_kv_heads], which the call keeps up (see
    ns_rope_append in the header for the format)."""
    n, width = qkv.shape
    row, one = qkv.stride()
    dtype = qkv.dtype
    assert width == (n_heads + 2 * n_kv_heads) * head_dim and (one == 1 or width == 1)
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise AssertionError("rope_append handles bfloat16 and float32")
    half = cos.shape[1]
    assert cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.shape == (n, half) and sin.shape == (n, half)
    assert cos.is_contiguous() and sin.is_contiguous() and 2 * half <= head_dim
    pool, n_slots, block_size, strides, code = _pool_args(dtype, n, n_kv_heads, head_dim, k_cache, v_cache, slots, k_scale, v_scale)
    dev = _lib.same_device(qkv, cos, sin, k_cache, v_cache, slots, k_scale, v_scale)
    q = qkv.new_empty(n, n_heads, head_dim)
    k = qkv.new_empty(n, n_kv_heads, head_dim) if dense_kv else None
    v = torch.empty_like(k) if dense_kv else None
    base, size = qkv.data_ptr(), 2 if dtype is torch.bfloat16 else 4
    base_k = base + n_heads * head_dim * size
    _lib.rope_append(dev, base, base_k, base_k + n_kv_heads * head_dim * size, row, row, row, cos.data_ptr(), sin.data_ptr(), 2 * half,
                     1 if interleaved else 0, q.data_ptr(), 0 if k is None else k.data_ptr(), 0 if v is None else v.data_ptr(), *pool, n, n_slots,
                     n_heads, n_kv_heads, head_dim, block_size, *strides, _lib.dtype_code(dtype), code)
    return q, k, v


def kv_append(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """rope_append without a rotation: store k_new / v_new [N, n_kv_heads, hd] (rotated already) at their slots."""
    assert k_new.dim() == 3 and v_new.shape == k_new.shape and k_new.dtype is v_new.dtype
    for t in (k_new, v_new):
        assert t.stride(2) == 1 and (t.shape[1] == 1 or t.stride(1) == t.shape[2]), "heads of a token must be adjacent"
    n, n_kv_heads, head_dim = k_new.shape
    dtype = k_new.dtype
    pool, n_slots, block_size, strides, code = _pool_args(dtype, n, n_kv_heads, head_dim, k_cache, v_cache, slots, k_scale, v_scale)
    dev = _lib.same_device(k_new, v_new, k_cache, v_cache, slots, k_scale, v_scale)
    _lib.rope_append(dev, 0, k_new.data_ptr(), v_new.data_ptr(), 0, k_new.stride(0), v_new.stride(0), 0, 0, 0, 0, 0, 0, 0, *pool, n, n_slots, 0,
                     n_kv_heads, head_dim, block_size, *strides, _lib.dtype_code(dtype), code)


def kv_values(pool: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values an int8 / float8_e4m3fn pool [blocks, block_size, n_kv_heads, hd] stands for under its scales, dense."""
    dev = _lib.same_device(pool, scale)
    code = _lib.kv8_code(pool.dtype)
    if code is None:
        raise NotImplementedError(f"kv_values reads int8 and float8_e4m3fn pools, not {pool.dtype}")
    assert pool.dim() == 4 and pool.stride(3) == 1
    strides = check_kv8_scales(pool, scale)
    out = scale.new_empty(*pool.shape) if dtype is torch.float32 else scale.new_empty(pool.shape, dtype=dtype)
    _lib.kv_values(dev, pool.data_ptr(), scale.data_ptr(), out.data_ptr(), *pool.shape, *pool.stride()[:3], *strides, _lib.dtype_code(dtype),
                   code)
    return out
