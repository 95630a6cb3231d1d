"""Engines on 8-bit KV pools and on scaled / partial / interleaved rotary positions, against a 64-bit emulation of the model."""
import pytest
import torch

from tests import kv8_reference as R
from tests.golden import make_golden as G

pytestmark = pytest.mark.gpu

CFG = dict(G.TINY_CFG, head_dim=64)          # a head size the tensor-core kernels take
YARN = {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
VARIANTS = {"plain": {}, "yarn": dict(rope_scaling=YARN), "partial-interleaved": dict(partial_rotary_factor=0.5, rope_interleaved=True)}


class Emulation:
    """One sequence's call through the Qwen2 layer stack in fp64. A code next to a rounding border may fall to either side of it
    (the engine's GEMMs are fp32, these are fp64), and such a step would grow from layer to layer: so every layer checks
    the rows that the engine's pool got against the exact ones, to within the format's half step, and goes on with the pool's."""

    def __init__(self, cfg, sd, pool):
        self.cfg, self.sd, self.pool = cfg, {k: v.double() for k, v in sd.items()}, pool

    def check_rows(self, vals, scale, exact, ctx):
        """vals [nb, bs, nkv, hd] of the sequence's blocks after the call, scale [nb, nkv], exact [T, nkv, hd] new rows."""
        bs, T = self.pool.block_size, exact.shape[0]
        pos = ctx + torch.arange(T)
        got = vals[pos // bs, pos % bs]
        slack = 1e-4 * exact.abs().max()                                      # fp32 GEMMs behind x
        if scale is None:
            assert bool(((got - exact).abs() <= slack).all())
            return
        s = scale[pos // bs][:, :, None].double()
        half = s / 2 if self.pool.kv_dtype == torch.int8 else torch.maximum(exact.abs() * 2.0 ** -4, s * 2.0 ** -10)
        assert bool(((got - exact).abs() <= half * (1 + 1e-4) + slack).all())
        q = R.QMAX[self.pool.kv_dtype]
        for blk in set((pos // bs).tolist()):
            if blk * bs >= ctx:                                               # the call wrote its first row: the scale is the call's
                top = exact[(pos // bs) == blk].abs().amax(dim=(0, 2))
                assert bool((top <= q * scale[blk] + slack).all()) and bool((top >= q * scale[blk] / 2 - slack).all())

    def feed(self, ids, ctx, blocks):
        """The call that put tokens `ids` on top of ctx stored ones, after the engine made it; logits of the last."""
        from nanoserve_b200.kernels.rotary import rotary_frequencies
        c, sd, pool = self.cfg, self.sd, self.pool
        T = len(ids)
        inv, f = rotary_frequencies(c.rotary_dim, c.rope_theta, c.rope_scaling)
        ang = (ctx + torch.arange(T)).double()[:, None] * inv.double()
        cos, sin = (f * ang.cos()).float(), (f * ang.sin()).float()
        norm = lambda x, w: w * x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + c.rms_norm_eps)
        x = sd["model.embed_tokens.weight"][torch.tensor(ids)]
        blk = torch.tensor(blocks[:-(-(ctx + T) // pool.block_size)])
        tables = torch.arange(len(blk))[None].int()
        for i in range(c.n_layers):
            p = f"model.layers.{i}."
            h = norm(x, sd[p + "input_layernorm.weight"])
            lin = lambda name: h @ sd[p + f"self_attn.{name}.weight"].t() + sd[p + f"self_attn.{name}.bias"]
            q, k, v = (R.f32(lin(n)).view(T, -1, c.head_dim) for n in ("q_proj", "k_proj", "v_proj"))
            q, k = R.rotate(q, cos, sin, c.rope_interleaved), R.rotate(k, cos, sin, c.rope_interleaved)
            vals = []
            for new, codes, scale in ((k, pool.k, pool.k_scale), (v, pool.v, pool.v_scale)):
                codes = codes[i].float().cpu()[blk].double()
                scale = None if scale is None else scale[i].cpu()[blk]
                vals.append(codes if scale is None else codes * scale.double()[:, None, :, None])
                self.check_rows(vals[-1], scale, new, ctx)
            o = R.attend_fast(q, vals[0], vals[1], tables, torch.tensor([ctx + T]), torch.tensor([0, T]), c.head_dim ** -0.5)
            x = x + o.reshape(T, -1) @ sd[p + "self_attn.o_proj.weight"].t()
            h = norm(x, sd[p + "post_attention_layernorm.weight"])
            g = h @ sd[p + "mlp.gate_proj.weight"].t()
            x = x + (g * torch.sigmoid(g) * (h @ sd[p + "mlp.up_proj.weight"].t())) @ sd[p + "mlp.down_proj.weight"].t()
        return norm(x, sd["model.norm.weight"])[-1] @ sd["model.embed_tokens.weight"].t()


def build(variant, kv_name, dtype=torch.float32, **kw):
    from nanoserve_b200.engine import LLMEngine
    from nanoserve_b200.model import ModelConfig, Qwen2Model
    sd = G.tiny_state_dict(CFG)
    cfg = ModelConfig(**dict(CFG, **VARIANTS[variant]))
    model = Qwen2Model(cfg, {k: v.to(dtype).cuda() for k, v in sd.items()})
    return cfg, sd, LLMEngine(model, eos_token_ids=[], kv_cache_dtype=kv_name, **dict(G.TINY_ENGINE_KW, **kw))


@pytest.mark.parametrize("variant", list(VARIANTS))
@pytest.mark.parametrize("kv_name", ["int8", "fp8_e4m3", None])
def test_engine_follows_the_emulation(variant, kv_name):
    """Several requests at once, prompts over block borders, chunked prefill, greedy steps from CUDA graphs."""
    if variant == "plain" and kv_name is None:
        pytest.skip("the 16-bit path has its own tests")
    cfg, sd, eng = build(variant, kv_name, max_num_batched_tokens=24)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 16, 41, 33)]
    ids = [eng.add_request(p, 12, ignore_eos=True) for p in prompts]
    toks = dict(zip(ids, [list(p) for p in prompts]))
    orig, steps = eng.scheduler.schedule, []

    def spy(now):
        plan = orig(now)
        steps[:] = [(s.seq_id, n, s.num_cached, list(s.block_table.blocks)) for s, n in zip(plan.scheduled, plan.chunks)]
        return plan

    eng.scheduler.schedule = spy
    em = Emulation(cfg, sd, eng.kv.pool)
    worst, sampled = 0.0, 0
    while eng.has_unfinished():
        outs = {o.seq_id: o.token for o in eng.step()}
        logits = eng.last_logits.double().cpu()
        for row, (sid, n, ctx, blocks) in enumerate(steps):
            want = em.feed(toks[sid][ctx:ctx + n], ctx, blocks)
            if sid in outs:
                worst = max(worst, (logits[row] - want).abs().max().item())
                toks[sid].append(outs[sid])
                sampled += 1
    assert sampled == 48 and eng.scheduler.num_preemptions == 0
    assert worst <= 1e-3, worst                     # the strict gate of this fp32 model


@pytest.mark.parametrize("kv_name", ["int8", "fp8_e4m3"])
def test_bf16_engine_with_prefix_hits_and_preemption(kv_name):
    """bf16, prefix caching and a pool so small that requests are preempted and recomputed: every request gets its tokens, the
    8-bit pool's logits stay near the 16-bit pool's on the same weights."""
    g = torch.Generator().manual_seed(4)
    kw = dict(prefix_caching=True, kv_cache_tokens=320, max_seq_len=128, max_num_seqs=6)
    cfg, sd, eng = build("plain", kv_name, torch.bfloat16, **kw)
    _, _, ref = build("plain", None, torch.bfloat16, **kw)
    head = torch.randint(0, cfg.vocab_size, (34,), generator=g).tolist()
    reqs = [head + torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (3, 9, 20, 1, 14, 6, 30, 8)]
    first = {}
    for e in (eng, ref):
        ids = [e.add_request(r, 40, ignore_eos=True) for r in reqs]
        out = {i: [] for i in ids}
        while e.has_unfinished():
            for o in e.step():
                out[o.seq_id].append(o.token)
        assert all(len(v) == 40 for v in out.values()) and e.buffers.device_errors == 0
        first[id(e)] = [out[i][0] for i in ids]
    assert eng.stats["prefix_hit_tokens"] > 0 and eng.stats["num_preemptions"] > 0
    assert eng.stats["kv_cache_dtype"] in ("int8", "float8_e4m3fn") and ref.stats["kv_cache_dtype"] == "bfloat16"
    assert eng.kv.pool.reserved_bytes < 0.6 * ref.kv.pool.reserved_bytes


def test_lookahead_and_sampling_run_on_an_8bit_pool():
    from nanoserve_b200.sampling import SamplingParams
    outs = []
    for lookahead in (False, True):
        _, _, eng = build("plain", "int8", torch.bfloat16, lookahead=lookahead)
        ids = [eng.add_request([1, 2, 3, 4 + i], 20, ignore_eos=True, sampling=SamplingParams(temperature=0.8, top_k=20, seed=i) if i else None)
               for i in range(4)]
        got = {i: [] for i in ids}
        while eng.has_unfinished():
            for o in eng.step():
                got[o.seq_id].append(o.token)
        outs.append([got[i] for i in ids])
    assert outs[0] == outs[1]


def test_speculative_engine_on_an_8bit_pool():
    """Rejected drafts rewind the tables and their rows are appended again: every request still gets its tokens."""
    from nanoserve_b200.model import ModelConfig, Qwen2Model
    from nanoserve_b200.speculative import SpeculativeEngine
    cfg = ModelConfig(**CFG)
    sd = {k: v.cuda() for k, v in G.tiny_state_dict(CFG).items()}
    target, draft = Qwen2Model(cfg, sd), Qwen2Model(cfg, {k: v + 0.02 * torch.randn_like(v) for k, v in sd.items()})
    eng = SpeculativeEngine(target, draft, [], num_speculative_tokens=3, max_seq_len=96, max_num_seqs=3, kv_cache_dtype="int8")
    ids = [eng.add_request([5, 6, 7 + i], 30, ignore_eos=True) for i in range(3)]
    got = {i: [] for i in ids}
    while eng.has_unfinished():
        for o in eng.step():
            got[o.seq_id].append(o.token)
    assert all(len(v) == 30 for v in got.values()) and eng.tpool.kv_dtype == torch.int8


def test_forward_batch_over_an_8bit_pool_fused_and_unfused():
    """The reference-style call over 8-bit pools, with fused and with unfused ops: both store the same rows up to half a step each
    (int8: s / 2 and the fp32 GEMMs' error), and answer."""
    from nanoserve_b200.kv_cache import PagedKVCache
    from nanoserve_b200.model import ModelConfig, Qwen2Model, SeqInput
    cfg = ModelConfig(**dict(CFG, **VARIANTS["partial-interleaved"]))
    sd = {k: v.cuda() for k, v in G.tiny_state_dict(CFG).items()}
    outs = []
    for fused in (True, False):
        m = Qwen2Model(cfg, dict(sd))
        m = m.with_fused_ops() if fused else m
        pool = PagedKVCache(cfg, 8, 16, "cuda", torch.float32, "int8")
        ids = torch.arange(3, 23, device="cuda")
        a = m.forward_batch(ids, torch.arange(20, device="cuda"), [SeqInput(20, block_table=[2, 5])], paged=pool,
                            slot_mapping=torch.cat((torch.arange(32, 48), torch.arange(80, 84))).cuda())
        k, v = pool.gather(0, torch.tensor([2, 5], device="cuda"), 20)
        assert k.shape == (1, cfg.n_kv_heads, 20, cfg.head_dim) and bool((k != 0).any())
        outs.append((a, k, pool.k_scale[0, [2, 5]].amax().item()))
    assert bool(torch.isfinite(outs[0][0]).all()) and outs[0][0].shape == outs[1][0].shape
    assert (outs[0][1] - outs[1][1]).abs().max().item() <= max(outs[0][2], outs[1][2]) * 1.001


def test_engine_refuses_unknown_cache_dtypes():
    with pytest.raises(ValueError):
        build("plain", "int4")
    with pytest.raises(ValueError):
        build("plain", "int8", block_size=24)
