"""8-bit KV pools and rotary positions: what is refused (before any launch), and the frequencies' formulas. No GPU."""
import ctypes
import math

import pytest
import torch

from nanoserve_b200 import _lib
from nanoserve_b200.kernels.rotary import check_kv8_scales, kv_values, rope_append, rope_tables, rotary_frequencies

P, NUL, F = ctypes.c_void_p, None, ctypes.c_float
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def msg():
    return _lib.load().ns_last_error().decode()


def rope_args(**kw):
    a = dict(q=P(256), k=P(512), v=P(1024), qs=1152, ks=1152, vs=1152, cos=P(2048), sin=P(4096), rot=64, inter=0, qo=P(8192), ko=NUL, vo=NUL,
             kp=P(16384), vp=P(32768), ksc=P(65536), vsc=P(131072), slots=P(262144), n=4, n_slots=1024, nh=14, nkv=2, hd=64, bs=16, sb=2048,
             sp=128, sh=64, scb=2, sch=1, dt=_lib.NS_BF16, pdt=_lib.NS_INT8, st=NUL)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def test_rope_append_refusals():
    f = _lib.load().ns_rope_append
    assert f(*rope_args(n=0)) == 0
    assert f(*rope_args(n=-1)) == INVALID
    assert f(*rope_args(rot=63)) == INVALID and "rotary dim 63" in msg()
    assert f(*rope_args(rot=66)) == INVALID
    assert f(*rope_args(cos=NUL)) == INVALID and "without tables" in msg()
    assert f(*rope_args(vp=NUL)) == INVALID and "both pools" in msg()
    assert f(*rope_args(slots=NUL)) == INVALID and "slots" in msg()
    assert f(*rope_args(vsc=NUL)) == INVALID and "scales" in msg()
    assert f(*rope_args(bs=24)) == UNSUPPORTED and "blocks of" in msg()
    assert f(*rope_args(bs=128)) == UNSUPPORTED
    assert f(*rope_args(dt=7)) == UNSUPPORTED
    assert f(*rope_args(pdt=_lib.NS_F32)) == UNSUPPORTED and "pool dtype" in msg()
    assert f(*rope_args(pdt=9)) == UNSUPPORTED
    assert f(*rope_args(k=NUL)) == INVALID and "null" in msg()


def attn_args(**kw):
    a = dict(q=P(256), k=P(512), v=P(1024), ks=P(2048), vs=P(4096), bt=P(8192), rows=NUL, lens=P(16384), cu=NUL, out=P(32768), S=2, N=2, nh=14,
             nkv=2, hd=64, bs=16, nb=64, tw=4, ts=4, qs=896, os=896, pb=2048, pp=128, ph=64, sb=2, sh=1, scale=F(0.125), dt=_lib.NS_BF16,
             pdt=_lib.NS_INT8, ws=NUL, wsb=0, wss=0, wst=0, st=NUL)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def test_attention_refusals():
    lib = _lib.load()
    f = lib.ns_ragged_paged_attn_q8
    simple = lambda **kw: lib.ns_ragged_paged_attn_q8_simple(*(attn_args(**kw)[:-5] + [NUL]))
    for call in (lambda **kw: f(*attn_args(**kw)), simple):
        assert call(S=0, N=0) == 0
        assert call(S=-1) == INVALID
        assert call(nh=15) == INVALID and "not divisible" in msg()
        assert call(dt=2) == UNSUPPORTED
        assert call(pdt=_lib.NS_BF16) == UNSUPPORTED and "8-bit" in msg()
        assert call(N=3) == INVALID and "one token" in msg()
        assert call(vs=NUL) == INVALID and "null" in msg()
        assert call(tw=-1) == INVALID
    assert simple(hd=300) == UNSUPPORTED and "head_dim" in msg()


def test_attention_workspace_refusals():
    lib = _lib.load()
    f = lambda **kw: lib.ns_ragged_paged_attn_q8(*attn_args(**kw))
    need = lib.ns_attn_workspace_bytes(2, 2, 14, 64)
    assert f(ws=NUL) == INVALID and "null" in msg()
    assert f(ws=P(4096 + 16), wsb=need, wss=2, wst=2) == INVALID and "aligned" in msg()
    assert f(ws=P(4096), wsb=need, wss=1, wst=2) == WORKSPACE and "exceeds" in msg()
    assert f(ws=P(4096), wsb=need, wss=2, wst=1) == WORKSPACE
    assert f(ws=P(4096), wsb=need - 1, wss=2, wst=2) == WORKSPACE and "needed" in msg()


def test_packed_calls():
    """The same checks behind ns_call, and its own: an operation it does not know, a wrong number of words, none at all."""
    import struct
    f = _lib.load().ns_call
    words = struct.pack("=2qd5q", 0, 0, 1.0, 0, 0, 1, 4, 0)
    assert f(0, words, 8) == INVALID and "null" in msg()
    assert f(0, words, 7) == INVALID and "takes 8 words, not 7" in msg()
    assert f(0, None, 8) == INVALID
    assert f(4, words, 8) == INVALID and "unknown operation 4" in msg() and f(-1, words, 8) == INVALID
    plain = [a.value if isinstance(a, (ctypes.c_void_p, ctypes.c_float)) else a or 0 for a in rope_args(bs=24)]
    assert f(1, struct.pack("=32q", *plain), 32) == UNSUPPORTED and "blocks of" in msg()
    plain = [a.value if isinstance(a, (ctypes.c_void_p, ctypes.c_float)) else a or 0 for a in attn_args(nh=15)]
    assert f(3, struct.pack("=26qd7q", *plain), 34) == INVALID and "15 heads not divisible" in msg()
    assert f(2, struct.pack("=15q", 256, 512, 1024, 2, 16, 2, 64, 2048, 128, 64, 2, 1, _lib.NS_INT8, _lib.NS_INT8, 0), 15) == UNSUPPORTED
    for op, count in ((_lib.rope_tables, 8), (_lib.rope_append, 32), (_lib.kv_values, 15), (_lib.ragged_paged_attn_q8, 34)):
        assert op.words == count == len(_lib.SIGNATURES[op.name][1])


def test_a_workspace_of_another_shape_is_refused():
    """Its counters lie elsewhere: they would be found non-zero."""
    from nanoserve_b200.kernels.paged_attention import AttnWorkspace, paged_attention_decode
    q, t, L = torch.zeros(2, 14, 64, dtype=torch.bfloat16), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    i8, s = torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(2, 2)
    for heads, hd in ((12, 64), (14, 128)):
        ws = AttnWorkspace(4, 4, heads, hd, device="cpu")
        with pytest.raises(ValueError, match="workspace"):
            paged_attention_decode(q, i8, i8, t, L, 0.125, workspace=ws, k_scale=s, v_scale=s)


def test_values_and_tables_refusals():
    lib = _lib.load()
    v = lambda dt, pdt, **kw: lib.ns_kv_values(P(256), kw.get("scale", P(512)), P(1024), kw.get("nb", 2), 16, 2, 64, 2048, 128, 64, 2, 1, dt, pdt, NUL)
    assert v(_lib.NS_BF16, _lib.NS_INT8, nb=0) == 0
    assert v(_lib.NS_INT8, _lib.NS_INT8) == UNSUPPORTED
    assert v(_lib.NS_F32, _lib.NS_F32) == UNSUPPORTED
    assert v(_lib.NS_F32, _lib.NS_E4M3, scale=NUL) == INVALID
    assert lib.ns_rope_tables(NUL, NUL, ctypes.c_double(1.0), NUL, NUL, 0, 4, NUL) == 0
    assert lib.ns_rope_tables(NUL, NUL, ctypes.c_double(1.0), NUL, NUL, 1, 4, NUL) == INVALID


def test_python_refusals():
    i8 = torch.zeros(2, 16, 2, 64, dtype=torch.int8)
    with pytest.raises(ValueError):
        check_kv8_scales(i8, None, None)
    with pytest.raises(AssertionError):
        check_kv8_scales(i8, torch.zeros(2, 3))
    with pytest.raises(AssertionError):
        check_kv8_scales(i8, torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.float64))
    with pytest.raises(_lib.NanoserveB200Error):
        kv_values(i8, torch.zeros(2, 2))
    with pytest.raises(_lib.NanoserveB200Error):
        rope_tables(torch.zeros(2, dtype=torch.int64), torch.ones(4))
    qkv, c = torch.zeros(3, 18 * 64, dtype=torch.bfloat16), torch.zeros(3, 32)
    with pytest.raises(_lib.NanoserveB200Error):
        rope_append(qkv, c, c, 14, 2, 64)
    with pytest.raises(AssertionError):
        rope_append(qkv, c[:2], c[:2], 14, 2, 64)
    with pytest.raises(AssertionError):
        rope_append(qkv.half(), c, c, 14, 2, 64)
    from nanoserve_b200.kernels.paged_attention import paged_attention_decode, ragged_paged_attention
    q, t, L = torch.zeros(2, 14, 64, dtype=torch.bfloat16), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(_lib.NanoserveB200Error):
        paged_attention_decode(q, i8, i8, t, L, 0.125, k_scale=torch.zeros(2, 2), v_scale=torch.zeros(2, 2))
    bf = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        ragged_paged_attention(q, bf, bf, t, L, None, 0.125, k_scale=torch.zeros(2, 2))


# ------------------------------------------------------------------------------------------------------ frequencies
def test_frequencies_default_linear_ntk():
    inv, f = rotary_frequencies(64, 1e6)
    want = [1e6 ** (-2 * i / 64) for i in range(32)]
    assert f == 1.0 and inv.dtype == torch.float32 and inv.tolist() == torch.tensor(want, dtype=torch.float64).float().tolist()
    lin, _ = rotary_frequencies(64, 1e6, {"type": "linear", "factor": 4.0})
    assert torch.equal(lin, inv / 4)                                            # a power of two: exact
    ntk, _ = rotary_frequencies(64, 1e4, {"rope_type": "ntk", "factor": 8.0})
    base, _ = rotary_frequencies(64, 1e4)
    assert ntk[0] == base[0] and abs(ntk[-1].item() * 8 / base[-1].item() - 1) < 2 ** -22


def test_frequencies_yarn():
    """Fast pairs keep their frequency, slow ones are divided by the factor, the ramp between is monotone."""
    sc = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    inv, f = rotary_frequencies(128, 1e6, sc)
    base, _ = rotary_frequencies(128, 1e6)
    ratio = inv.double() / base.double()
    turns = 32768 * base.double() / (2 * math.pi)
    assert abs(f - (0.1 * math.log(4.0) + 1.0)) < 1e-12
    assert bool((ratio[turns > 40] == 1.0).all()) and bool(((ratio[turns < 0.8] - 0.25).abs() < 2 ** -23).all())
    assert bool((ratio[1:] <= ratio[:-1] + 2 ** -22).all())
    assert rotary_frequencies(128, 1e6, dict(sc, attention_factor=1.5))[1] == 1.5


@pytest.mark.parametrize("bad", [dict(rotary_dim=63), dict(rotary_dim=0), dict(theta=0.5), dict(scaling={"type": "linear", "factor": 0.5}),
                                 dict(scaling={"type": "yarn", "factor": 2.0}), dict(rotary_dim=2, scaling={"type": "ntk", "factor": 2.0})])
def test_frequencies_refusals(bad):
    args = dict(rotary_dim=64, theta=1e4, scaling=None)
    args.update(bad)
    with pytest.raises(ValueError):
        rotary_frequencies(**args)


def test_unknown_scaling_type():
    with pytest.raises(NotImplementedError):
        rotary_frequencies(64, 1e4, {"type": "other", "factor": 2.0})


# ------------------------------------------------------------------------------------------------------ pool and configuration
def tiny_cfg(**kw):
    from nanoserve_b200.model import ModelConfig
    return ModelConfig(**dict(dict(vocab_size=8, hidden_size=8, n_layers=3, n_heads=2, n_kv_heads=2, head_dim=64, intermediate_size=8,
                                   rope_theta=1e4, rms_norm_eps=1e-6, tie_word_embeddings=True), **kw))


def test_pool_of_8bit_codes():
    from nanoserve_b200.kv_cache import PagedKVCache, kv_cache_bytes_per_block, resolve_kv_dtype
    cfg = tiny_cfg()
    for name, dt in (("int8", torch.int8), ("fp8_e4m3", torch.float8_e4m3fn), (torch.int8, torch.int8)):
        pool = PagedKVCache(cfg, 5, 16, "cpu", torch.bfloat16, name)
        assert pool.k.dtype == dt and pool.k.shape == (3, 5, 16, 2, 64) and pool.k_scale.shape == (3, 5, 2)
        assert pool.reserved_bytes == pool.k.numel() * 2 + pool.k_scale.numel() * 8
        assert pool.scales(1)["v_scale"].data_ptr() == pool.v_scale[1].data_ptr()
    plain = PagedKVCache(cfg, 5, 16, "cpu", torch.bfloat16)
    assert plain.kv_dtype is None and plain.scales(0) == {} and plain.reserved_bytes == plain.k.numel() * 4
    per = kv_cache_bytes_per_block(cfg, 16, torch.bfloat16, "int8")
    assert PagedKVCache.tokens_for_bytes(cfg, 10 * per + 5, torch.bfloat16, "int8") == 160
    assert PagedKVCache.tokens_for_bytes(cfg, 10 * per, torch.bfloat16) == 10 * per // cfg.kv_bytes_per_token(torch.bfloat16)
    assert resolve_kv_dtype("auto") is None
    for bad in ("int4", torch.float16, 8):
        with pytest.raises(ValueError):
            resolve_kv_dtype(bad)
    with pytest.raises(ValueError):
        PagedKVCache(cfg, 5, 24, "cpu", torch.bfloat16, "int8")


def test_configuration_of_rotary_positions():
    from nanoserve_b200.model import ModelConfig
    assert tiny_cfg().plain_rope and tiny_cfg().rotary_dim == 64
    assert not tiny_cfg(partial_rotary_factor=0.5).plain_rope and tiny_cfg(partial_rotary_factor=0.4).rotary_dim == 24
    assert not tiny_cfg(rope_interleaved=True).plain_rope and tiny_cfg(rope_scaling={"type": "default"}).plain_rope
    hf = dict(vocab_size=8, hidden_size=128, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, intermediate_size=8,
              rms_norm_eps=1e-6, rope_theta=1e6)
    yarn = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    assert ModelConfig.from_hf_config(hf).plain_rope
    scaled = dict(hf, rope_scaling=yarn, partial_rotary_factor=0.5)
    assert ModelConfig.from_hf_config(scaled) == ModelConfig.from_hf_config(hf)          # as before there were such positions
    cfg = ModelConfig.from_hf_config(scaled, rope_extensions=True)
    assert cfg.rope_scaling == yarn and cfg.rotary_dim == 32 and hash(cfg) == hash(cfg)
    new = ModelConfig.from_hf_config(dict({k: v for k, v in hf.items() if k != "rope_theta"},
                                          rope_parameters=dict(rope_type="linear", factor=2.0, rope_theta=5e5, partial_rotary_factor=0.5)), True)
    assert new.rope_theta == 5e5 and new.rotary_dim == 32 and new.rope_scaling["factor"] == 2.0
    assert ModelConfig.from_hf_config(dict(hf, rope_parameters=dict(rope_type="default", rope_theta=1e6)), True).plain_rope
