"""Ragged paged attention on sm_100a.

`paged_attention_decode` keeps the name and signature of the reference's Triton wrapper
(nanoserve/kernels/paged_attention.py:85-105). `ragged_paged_attention` is the single call that replaces the
whole of nanoserve/model.py:262-323 (`Qwen2Model._attend`): decode rows and prefill chunks of a mixed step in
one pass over the paged pool, driven by block_tables / seq_lens / cu_seqlens that live on the device.

The tensor-core kernels need a small caller-owned workspace (`AttnWorkspace`): it holds the per-step plan
(built once per step by `plan`, reused by every layer) and the split-KV partials. Convenience calls without
an explicit workspace use a cached one per device.
"""
from __future__ import annotations

import torch

from nanoserve_b200 import _lib
from nanoserve_b200.kernels.rotary import check_kv8_scales


class AttnWorkspace:
    """Zero-initialised device buffer sized for up to max_seqs sequences / max_tokens query tokens."""

    def __init__(self, max_seqs: int, max_tokens: int, n_heads: int, head_dim: int, device="cuda"):
        self.max_seqs, self.max_tokens = int(max_seqs), int(max(max_tokens, max_seqs))
        self.n_heads, self.head_dim = n_heads, head_dim
        nbytes = _lib.load().ns_attn_workspace_bytes(self.max_seqs, self.max_tokens, n_heads, head_dim)
        if nbytes <= 0:
            raise _lib.NanoserveB200Error("ns_attn_workspace_bytes rejected the sizes")
        self.nbytes = int(nbytes)
        # +256 so the used part can start on a 256-byte boundary whatever the allocator returns
        self._raw = torch.zeros(self.nbytes + 256, dtype=torch.uint8, device=device)
        off = (-self._raw.data_ptr()) % 256
        self.buf = self._raw[off:off + self.nbytes]
        self.ptr = self.buf.data_ptr()

    def fits(self, n_seqs: int, n_tokens: int, n_heads: int, head_dim: int) -> bool:
        return (n_seqs <= self.max_seqs and n_tokens <= self.max_tokens and n_heads == self.n_heads
                and head_dim == self.head_dim)

    def plan(self, seq_lens: torch.Tensor, cu_seqlens: torch.Tensor | None, n_seqs: int, block_size: int,
             table_rows: torch.Tensor | None = None) -> None:
        """Build this step's plan (call once per step, before the first layer's attention)."""
        _lib.call("ns_attn_plan", seq_lens.data_ptr(), _lib.ptr(cu_seqlens), _lib.ptr(table_rows), n_seqs, block_size,
                  self.n_heads,
                  self.head_dim, self.buf.data_ptr(), self.nbytes, self.max_seqs, self.max_tokens, _lib.stream_ptr())


_cached: dict[tuple, AttnWorkspace] = {}
_cached_q8: dict[tuple, AttnWorkspace] = {}


def _workspace_q8(device, n_seqs: int, n_tokens: int, n_heads: int, head_dim: int) -> AttnWorkspace:
    """The workspace of a call over an 8-bit pool that brings none: one per device and stream, so that calls on two streams
    never share one; inside a graph capture a new one, which belongs to the graph."""
    if torch.cuda.is_current_stream_capturing():
        return AttnWorkspace(max(n_seqs, 1), max(n_tokens, 1), n_heads, head_dim, device)
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index), n_heads, head_dim)
    ws = _cached_q8.get(key)
    if ws is None or n_seqs > ws.max_seqs or n_tokens > ws.max_tokens:
        cap_s, cap_t = max(256, 1 << (max(n_seqs, 1) - 1).bit_length()), max(4096, 1 << (max(n_tokens, 1) - 1).bit_length())
        ws = _cached_q8[key] = AttnWorkspace(cap_s, cap_t, n_heads, head_dim, device)
    return ws


def _workspace_for(device, n_seqs: int, n_tokens: int, n_heads: int, head_dim: int) -> AttnWorkspace:
    key = (device.index if device.index is not None else torch.cuda.current_device(), n_heads, head_dim)
    ws = _cached.get(key)
    if ws is None or not ws.fits(n_seqs, n_tokens, n_heads, head_dim):
        cap_s = max(256, 1 << (max(n_seqs, 1) - 1).bit_length())
        cap_t = max(4096, 1 << (max(n_tokens, 1) - 1).bit_length())
        ws = _cached[key] = AttnWorkspace(cap_s, cap_t, n_heads, head_dim, device)
    return ws


def _check_pool(q, k_pool, v_pool):
    assert k_pool.dim() == 4 and q.dim() == 3
    assert q.stride(-1) == 1 and k_pool.stride(-1) == 1 and v_pool.stride() == k_pool.stride()
    assert q.stride(1) == q.shape[2], "query heads must be adjacent (head stride == head_dim)"
    assert k_pool.dtype == q.dtype and v_pool.dtype == q.dtype


def _attend_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, table_rows, seq_lens, cu_seqlens, scale, n_seqs, ws, planned, out,
               simple) -> torch.Tensor:
    """Ragged attention over an int8 / float8_e4m3fn pool (ns_ragged_paged_attn_q8). (A decode step makes one such call per layer:
    the checks look at every tensor once.)"""
    N, n_heads, head_dim = q.shape
    pool_shape = num_blocks, block_size, n_kv_heads, hd = k_pool.shape
    rows, width = block_tables.shape
    q0, q1, q2 = q.stride()
    ps = p0, p1, p2, p3 = k_pool.stride()
    t0, t1 = block_tables.stride()
    i32, kv_dtype, q_dtype = torch.int32, k_pool.dtype, q.dtype
    if v_scale is None:
        raise ValueError(f"a {kv_dtype} pool needs k_scale and v_scale (fp32 [num_blocks, n_kv_heads])")
    s0, s1 = check_kv8_scales(k_pool, k_scale, v_scale)
    assert hd == head_dim and p3 == 1 and v_pool.shape == pool_shape and v_pool.stride() == ps and v_pool.dtype is kv_dtype
    assert q2 == 1 and (q1 == head_dim or n_heads == 1), "query heads must be adjacent (head stride == head_dim)"
    assert block_tables.dtype is i32 and (t1 == 1 or width <= 1)
    assert seq_lens.dtype is i32 and seq_lens.is_contiguous() and seq_lens.shape[0] >= n_seqs
    if ws is not None and (ws.n_heads != n_heads or ws.head_dim != head_dim):
        raise ValueError(f"a workspace for {ws.n_heads} heads of {ws.head_dim} does not serve {n_heads} heads of {head_dim}")
    dev = _lib.same_device(q, k_pool, v_pool, k_scale, v_scale, block_tables, seq_lens, None if ws is None else ws.buf)
    cu = rows_ptr = 0
    if cu_seqlens is None:
        assert N == n_seqs, "without cu_seqlens every sequence has one token"
    else:
        assert cu_seqlens.dtype is i32 and cu_seqlens.is_contiguous() and cu_seqlens.shape[0] > n_seqs
        cu = cu_seqlens.data_ptr()
        _lib.same_device(q, cu_seqlens)
    if table_rows is None:
        assert rows >= n_seqs, "block_tables has a row per sequence"
    else:
        assert table_rows.dtype is i32 and table_rows.is_contiguous() and table_rows.shape[0] >= n_seqs
        rows_ptr = table_rows.data_ptr()
        _lib.same_device(q, table_rows)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
        o0 = n_heads * head_dim
    else:
        o0, o1, o2 = out.stride()
        assert out.shape == q.shape and o2 == 1 and (o1 == head_dim or n_heads == 1) and out.dtype is q_dtype
        _lib.same_device(q, out)
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):                       # a launch needs its device current
            return _attend_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, table_rows, seq_lens, cu_seqlens, scale, n_seqs, ws, planned,
                              out, simple)
    args = (q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_tables.data_ptr(), rows_ptr,
            seq_lens.data_ptr(), cu, out.data_ptr(), n_seqs, N, n_heads, n_kv_heads, head_dim, block_size, num_blocks, width, t0, q0, o0, p0, p1,
            p2, s0, s1, scale, _lib.dtype_code(q_dtype), _lib.kv8_code(kv_dtype))
    if simple:
        _lib.call("ns_ragged_paged_attn_q8_simple", *args, torch._C._cuda_getCurrentRawStream(dev))
        return out
    if ws is None:
        ws = _workspace_q8(q.device, n_seqs, N, n_heads, head_dim)
    if cu and N > 1:
        if not planned:
            ws.plan(seq_lens, cu_seqlens, n_seqs, block_size, table_rows)
        _lib.note_launches(1)          # the prefill-tile kernel is launched next to the decode kernel
    _lib.ragged_paged_attn_q8(dev, *args, ws.ptr, ws.nbytes, ws.max_seqs, ws.max_tokens)
    return out


def paged_attention_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, scale: float, workspace: AttnWorkspace | None = None,
                           k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """q: [B, n_heads, head_dim]; k_pool/v_pool: ONE layer's pool [num_blocks, block_size, n_kv_heads, head_dim];
    block_tables: int32 [B, max_blocks]; context_lens: int32 [B] (includes the new token, whose K/V must already
    be written). An int8 / float8_e4m3fn pool comes with k_scale / v_scale, fp32 [num_blocks, n_kv_heads] (q may then be
    bf16 or fp32). Returns [B, n_heads, head_dim]."""
    if _lib.kv8_code(k_pool.dtype) is not None:
        return _attend_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, None, context_lens, None, scale, q.shape[0], workspace, False,
                          None, False)
    assert k_scale is None and v_scale is None, "scales belong to 8-bit pools"
    _lib.require_cuda(q, k_pool, v_pool, block_tables, context_lens)
    _check_pool(q, k_pool, v_pool)
    assert block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32
    assert block_tables.stride(-1) == 1 and context_lens.is_contiguous()
    B, n_heads, head_dim = q.shape
    _, block_size, n_kv_heads, _ = k_pool.shape
    out = torch.empty(B, n_heads, head_dim, device=q.device, dtype=q.dtype)
    ws = workspace or _workspace_for(q.device, B, B, n_heads, head_dim)
    _lib.call("ns_paged_attn_decode", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(),
              context_lens.data_ptr(), out.data_ptr(), B, n_heads, n_kv_heads, head_dim, block_size,
              block_tables.stride(0), q.stride(0), out.stride(0), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2),
              float(scale), _lib.dtype_code(q.dtype), ws.buf.data_ptr(), ws.nbytes, ws.max_seqs, ws.max_tokens,
              _lib.stream_ptr())
    return out


def paged_attention_decode_static(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                                  block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                                  out: torch.Tensor) -> torch.Tensor:
    """paged_attention_decode for callers that may not allocate on the device: `out` is supplied by the caller and
    the kernels' scratch is a fixed array inside the library (no workspace tensor, no torch allocation here).
    Limits: at most 64 rows, 32 query heads, head_dim 64 or 128, bf16, block size 16; larger inputs raise. All
    calls on a GPU share that scratch, so keep them on one stream; make the first call on each device outside any
    CUDA-graph capture (it resolves the scratch address)."""
    _lib.require_cuda(q, k_pool, v_pool, block_tables, context_lens, out)
    _check_pool(q, k_pool, v_pool)
    assert block_tables.dtype == torch.int32 and context_lens.dtype == torch.int32
    assert block_tables.stride(-1) == 1 and context_lens.is_contiguous()
    assert out.shape == q.shape and out.dtype == q.dtype and out.stride(-1) == 1 and out.stride(1) == q.shape[2]
    B, n_heads, head_dim = q.shape
    _, block_size, n_kv_heads, _ = k_pool.shape
    _lib.call("ns_paged_attn_decode_static", q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(),
              context_lens.data_ptr(), out.data_ptr(), B, n_heads, n_kv_heads, head_dim, block_size,
              block_tables.stride(0), q.stride(0), out.stride(0), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2),
              float(scale), _lib.dtype_code(q.dtype), _lib.stream_ptr())
    return out


def ragged_paged_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                           seq_lens: torch.Tensor, cu_seqlens: torch.Tensor | None, scale: float, *,
                           n_seqs: int | None = None, table_rows: torch.Tensor | None = None,
                           workspace: AttnWorkspace | None = None, planned: bool = False,
                           out: torch.Tensor | None = None, simple: bool = False, k_scale: torch.Tensor | None = None,
                           v_scale: torch.Tensor | None = None) -> torch.Tensor:
    """Attention for a mixed step. q: [N, n_heads, head_dim] = the flattened query tokens of S sequences;
    sequence s owns rows cu_seqlens[s]..cu_seqlens[s+1]-1 and seq_lens[s] keys (context + its new tokens,
    already in the pool), reached through block_tables[table_rows[s] if given else s]. cu_seqlens=None means
    one token per sequence. `planned=True` says workspace.plan(...) was already called for this step (the
    per-layer fast path); otherwise the plan is built here. `simple=True` forces the scalar fp32-accumulating
    kernel. An int8 / float8_e4m3fn pool comes with k_scale / v_scale, fp32 [num_blocks, n_kv_heads]; q is then bf16 or
    fp32, and a plan is needed only when some sequence has more than one token. Returns [N, n_heads, head_dim]."""
    if _lib.kv8_code(k_pool.dtype) is not None:
        return _attend_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, table_rows, seq_lens, cu_seqlens, scale,
                          int(n_seqs) if n_seqs is not None else seq_lens.shape[0], workspace, planned, out, simple)
    assert k_scale is None and v_scale is None, "scales belong to 8-bit pools"
    _lib.require_cuda(q, k_pool, v_pool, block_tables, seq_lens, cu_seqlens, table_rows)
    _check_pool(q, k_pool, v_pool)
    assert block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32 and block_tables.stride(-1) == 1
    assert cu_seqlens is None or (cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous())
    assert table_rows is None or (table_rows.dtype == torch.int32 and table_rows.is_contiguous())
    N, n_heads, head_dim = q.shape
    S = int(n_seqs) if n_seqs is not None else seq_lens.shape[0]
    _, block_size, n_kv_heads, _ = k_pool.shape
    if out is None:
        out = torch.empty(N, n_heads, head_dim, device=q.device, dtype=q.dtype)
    else:
        assert out.shape == q.shape and out.stride(-1) == 1 and out.stride(1) == head_dim and out.dtype == q.dtype
    code = _lib.dtype_code(q.dtype)
    common = (q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), block_tables.data_ptr(), _lib.ptr(table_rows),
              seq_lens.data_ptr(), _lib.ptr(cu_seqlens), out.data_ptr(), S, N, n_heads, n_kv_heads, head_dim, block_size,
              block_tables.stride(0), q.stride(0), out.stride(0), k_pool.stride(0), k_pool.stride(1), k_pool.stride(2),
              float(scale), code)
    if simple or code != _lib.NS_BF16:
        _lib.call("ns_ragged_paged_attn_simple", *common, _lib.stream_ptr())
        return out
    ws = workspace or _workspace_for(q.device, S, N, n_heads, head_dim)
    if not planned:
        ws.plan(seq_lens, cu_seqlens, S, block_size, table_rows)
    _lib.call("ns_ragged_paged_attn", *common, ws.buf.data_ptr(), ws.nbytes, ws.max_seqs, ws.max_tokens,
              _lib.stream_ptr())
    if cu_seqlens is not None and N > S:
        _lib.note_launches(1)          # the prefill-tile kernel is launched next to the decode kernel
    return out
