"""Rotary tables, rotation + append (16/32-bit and 8-bit pools) and attention over 8-bit pools, against 64-bit plain forms."""
import math

import pytest
import torch

from tests import kv8_reference as R

pytestmark = pytest.mark.gpu

KV8 = [torch.int8, torch.float8_e4m3fn]
BS = 16


def tables_for(positions, rot, theta=1e6):
    from nanoserve_b200.kernels.rotary import rope_tables, rotary_frequencies
    inv, f = rotary_frequencies(rot, theta)
    return rope_tables(positions.cuda(), inv.cuda(), f)


# ------------------------------------------------------------------------------------------------------ tables
@pytest.mark.parametrize("far", [1, 5000, 131072, 10_000_000, 2 ** 40])
@pytest.mark.parametrize("half", [1, 10, 32, 64])
def test_tables_are_exact_to_fp32_at_any_position(far, half):
    from nanoserve_b200.kernels.rotary import rope_tables
    g = torch.Generator().manual_seed(half)
    pos = torch.randint(0, far, (37,), generator=g)
    pos[0], pos[1] = 0, far - 1
    inv = (1e4 ** (-torch.arange(half).double() / max(half, 1))).float()
    cos, sin = rope_tables(pos.cuda(), inv.cuda(), 1.25)
    ang = pos.double()[:, None] * inv.double()
    # one rounding to fp32 (2^-24 of the value); the fp64 angle (three roundings of 2^-53) may be off by its own size times that,
    # in the kernel and in the reference alike
    for got, want in ((cos, 1.25 * ang.cos()), (sin, 1.25 * ang.sin())):
        tol = 2.0 ** -24 * want.abs() + 1.25 * (8 * 2.0 ** -53) * ang.abs() + 2.0 ** -50
        assert bool(((got.cpu().double() - want).abs() <= tol).all())


def test_tables_of_no_tokens_and_no_pairs():
    from nanoserve_b200.kernels.rotary import rope_tables
    c, s = rope_tables(torch.empty(0, dtype=torch.int64, device="cuda"), torch.ones(4, device="cuda"))
    assert c.shape == (0, 4) and s.shape == (0, 4)
    c, _ = rope_tables(torch.zeros(3, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda"))
    assert c.shape == (3, 0)


# ------------------------------------------------------------------------------------------------------ rotation, 16/32-bit pools
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,rot", [(14, 2, 64, 64), (14, 2, 64, 32), (12, 2, 128, 128), (5, 1, 128, 48), (3, 3, 80, 20), (4, 2, 64, 0),
                                           (2, 1, 36, 36), (9, 3, 256, 64), (6, 2, 64, 24)])
def test_rope_append_16bit_is_the_definition(nh, nkv, hd, rot, interleaved, dtype):
    from nanoserve_b200.kernels.rotary import rope_append
    g = torch.Generator().manual_seed(nh * hd + rot)
    N, nb = 23, 9
    wide = (torch.randn(N, (nh + 2 * nkv) * hd + 8, generator=g)).to(dtype)
    qkv = wide[:, :(nh + 2 * nkv) * hd]                                        # strided rows
    cos, sin = tables_for(torch.randint(0, 100000, (N,), generator=g), rot) if rot else (torch.empty(N, 0).cuda(),) * 2
    slots = torch.randperm(nb * BS, generator=g)[:N]
    slots[3], slots[7] = -1, nb * BS                                            # stored nowhere
    kp, vp = [torch.randn(nb, BS, nkv, hd, generator=g).to(dtype) for _ in range(2)]
    kc, vc = kp.cuda(), vp.cuda()
    q, k, v = rope_append(wide.cuda()[:, :qkv.shape[1]], cos, sin, nh, nkv, hd, kc, vc, slots.cuda(), interleaved=interleaved, dense_kv=True)
    x = qkv.double().view(N, nh + 2 * nkv, hd)
    rot64 = R.rotate(x[:, :nh + nkv], cos.cpu(), sin.cpu(), interleaved).to(dtype)
    assert torch.equal(q.cpu(), rot64[:, :nh]) and torch.equal(k.cpu(), rot64[:, nh:])
    assert torch.equal(v.cpu(), x[:, nh + nkv:].to(dtype))
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < nb * BS:
            kp.view(-1, nkv, hd)[s], vp.view(-1, nkv, hd)[s] = rot64[t, nh:], x[t, nh + nkv:].to(dtype)
    assert torch.equal(kc.cpu(), kp) and torch.equal(vc.cpu(), vp)


def test_rope_append_agrees_with_rope_qkv_where_both_apply():
    """fp32, half layout, whole head: the table entries are the only difference between the two, and these are equal here."""
    from nanoserve_b200.kernels.fused import rope_qkv
    from nanoserve_b200.kernels.rotary import rope_append
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(17, (14 + 4) * 64, generator=g).cuda()
    cos, sin = tables_for(torch.arange(17), 64)
    a = rope_append(qkv, cos, sin, 14, 2, 64, dense_kv=True)
    b = rope_qkv(qkv, torch.cat((cos, cos), 1), torch.cat((sin, sin), 1), 14, 2, 64)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------------ append, 8-bit pools
def random_pool(g, nb, bs, nkv, hd, kv, spread=1.0):
    x = torch.randn(nb, bs, nkv, hd, generator=g).double() * spread
    s = torch.tensor([[R.pow2_scale(x[b, :, h].abs().max().item(), R.QMAX[kv]) for h in range(nkv)] for b in range(nb)])
    codes = R.encode(x / s.double()[:, None, :, None], kv).float()
    return codes.to(kv), s.float()


def run_append(qkv, cos, sin, nh, nkv, hd, pools, slots, interleaved=False):
    from nanoserve_b200.kernels.rotary import rope_append
    (kp, ks), (vp, vs) = pools
    dev = [t.cuda() for t in (kp, ks, vp, vs)]
    q, _, _ = rope_append(qkv.cuda(), cos, sin, nh, nkv, hd, dev[0], dev[2], slots.cuda(), k_scale=dev[1], v_scale=dev[3],
                          interleaved=interleaved)
    return q.cpu(), [t.cpu() for t in dev]


def check_append(qkv, cos, sin, nh, nkv, hd, pools, slots, interleaved=False):
    N = qkv.shape[0]
    q, (kc, ks, vc, vs) = run_append(qkv, cos, sin, nh, nkv, hd, pools, slots, interleaved)
    x = qkv.double().view(N, nh + 2 * nkv, hd)
    rot = R.rotate(x[:, :nh + nkv], cos.cpu(), sin.cpu(), interleaved)
    assert torch.equal(q, rot[:, :nh].to(qkv.dtype))
    for (pool, scale), got_c, got_s, vals in ((pools[0], kc, ks, rot[:, nh:]), (pools[1], vc, vs, x[:, nh + nkv:])):
        want_c, want_s = R.append(pool, scale, vals, slots.tolist())
        wrong = int((torch.nan_to_num(got_s.double(), nan=-1.0) != torch.nan_to_num(want_s, nan=-1.0)).sum())
        assert wrong == 0, f"{wrong} scales differ"
        wrong = (got_c.float().double() != want_c).nonzero().tolist()
        assert not wrong, f"{len(wrong)} codes differ, the first at {wrong[0]}"


@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,rot,bs,interleaved", [(14, 2, 64, 64, 16, False), (12, 2, 128, 64, 16, True), (4, 1, 80, 20, 16, False),
                                                          (3, 3, 36, 36, 8, True), (8, 8, 128, 128, 32, False), (2, 2, 256, 32, 64, False),
                                                          (5, 1, 64, 0, 1, False)])
def test_append8_is_the_definition(nh, nkv, hd, rot, bs, interleaved, dtype, kv):
    """Sequences that re-open a part-filled block, chunks that start inside one and run over several, fresh blocks, strays."""
    g = torch.Generator().manual_seed(hd + rot + bs)
    starts = [(3 % bs, 1), (0, 1), (bs - 1, 1), (5 % bs, 2 * bs + 3), (0, 3 * bs), (bs // 2, 1)]
    nb = sum((c + t - 1) // bs + 1 for c, t in starts) + 3
    perm = torch.randperm(nb, generator=g)
    slots, used = [], 0
    for c, t in starts:
        p = torch.arange(c, c + t)
        slots.append(perm[used + p // bs] * bs + p % bs)
        used += (c + t - 1) // bs + 1
    slots = torch.cat(slots + [torch.tensor([-1, nb * bs, -(2 ** 40), 2 ** 40])])
    N = slots.shape[0]
    qkv = (torch.randn(N, (nh + 2 * nkv) * hd, generator=g) * 2).to(dtype)
    cos, sin = tables_for(torch.randint(0, 100000, (N,), generator=g), rot) if rot else (torch.empty(N, 0).cuda(),) * 2
    pools = [random_pool(g, nb, bs, nkv, hd, kv, s) for s in (0.7, 1.3)]
    check_append(qkv, cos, sin, nh, nkv, hd, pools, slots, interleaved)


@pytest.mark.parametrize("kv", KV8)
def test_append8_tokens_in_any_order_and_slots_named_twice(kv):
    """One owner per block: shuffled tokens, two separate runs into one block, and the later of two tokens with one slot."""
    g = torch.Generator().manual_seed(5)
    nkv, hd, nb, N = 2, 64, 6, 90
    slots = torch.randint(0, nb * BS, (N,), generator=g)                      # far more tokens than slots of a block
    slots[40:60] = 7                                                          # as graph padding does: one slot, many times
    qkv = torch.randn(N, 3 * nkv * hd, generator=g).bfloat16()
    cos, sin = tables_for(torch.arange(N), hd)
    check_append(qkv, cos, sin, nkv, nkv, hd, [random_pool(g, nb, BS, nkv, hd, kv) for _ in range(2)], slots)


@pytest.mark.parametrize("kv", KV8)
def test_append8_many_tokens_spread_over_many_ctas(kv):
    """More than 1024 tokens (the larger token pieces), blocks whose tokens lie in different pieces."""
    g = torch.Generator().manual_seed(6)
    nkv, hd, nb, N = 1, 64, 90, 1400
    slots = torch.randperm(nb * BS, generator=g)[:N]
    slots[::2] = slots[::2].sort().values
    qkv = torch.randn(N, 3 * nkv * hd, generator=g).bfloat16()
    cos, sin = tables_for(torch.arange(N), hd)
    check_append(qkv, cos, sin, nkv, nkv, hd, [random_pool(g, nb, BS, nkv, hd, kv) for _ in range(2)], slots)


@pytest.mark.parametrize("kv", KV8)
def test_append8_extreme_values(kv):
    """Zero rows, magnitudes at the code range's border (127 s and 448 s exactly and just above), tiny and huge ones,
    infinities and NaN (their block and head reads as NaN, its neighbours do not), a scale of zero."""
    g = torch.Generator().manual_seed(7)
    nkv, hd, nb = 2, 64, 12
    q = R.QMAX[kv]
    tops = [0.0, q, math.nextafter(q, 1e9), q / 2 ** 20, 1e-38, 1e-45, 3.0e38, float("inf"), float("nan"), 1.0, 0.3]
    N = len(tops)
    qkv = torch.randn(N, 3 * nkv * hd, generator=g)
    x = qkv.view(N, 3 * nkv, hd)
    for t, top in enumerate(tops):
        for h in (nkv, 2 * nkv):
            if not math.isnan(top) and top < 1e30:
                x[t, h] *= min(top, 1.0) / 8
            x[t, h, 5] = torch.tensor(top, dtype=torch.float64).float()
    slots = torch.tensor([b * BS + (0 if b % 2 else 4) for b in range(N)])
    pools = [random_pool(g, nb, BS, nkv, hd, kv) for _ in range(2)]
    pools[0][1][0] = 0.0
    pools[1][1][2] = float("nan")
    pools[1][1][4] = 0.037                                                     # another writer's scale: no power of two
    cos, sin = torch.empty(N, 0).cuda(), torch.empty(N, 0).cuda()
    check_append(qkv, cos, sin, nkv, nkv, hd, pools, slots)


def test_append8_one_by_one_equals_in_one_go():
    """e4m3 codes survive a growing scale: a block filled token by token stands for what one call would have stored."""
    from nanoserve_b200.kernels.rotary import kv_append, kv_values
    g = torch.Generator().manual_seed(8)
    x = (torch.randn(BS, 1, 64, generator=g) * torch.linspace(0.5, 40, BS)[:, None, None]).cuda()
    pools = []
    for steps in ([BS], [1] * BS, [5, 1, 10]):
        kc, vc = [torch.zeros(1, BS, 1, 64, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
        ks, vs = [torch.zeros(1, 1, device="cuda") for _ in range(2)]
        a = 0
        for n in steps:
            kv_append(x[a:a + n], x[a:a + n], kc, vc, torch.arange(a, a + n, device="cuda"), ks, vs)
            a += n
        pools.append(kv_values(kc, ks))
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])


@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 20])
def test_kv_values(kv, dtype, hd):
    from nanoserve_b200.kernels.rotary import kv_values
    g = torch.Generator().manual_seed(9)
    pool, scale = random_pool(g, 5, BS, 3, hd, kv)
    view = pool.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)         # heads outside positions
    got = kv_values(view, scale.cuda(), dtype)
    assert torch.equal(got.cpu(), R.values(pool, scale).to(dtype))


# ------------------------------------------------------------------------------------------------------ attention
CONFIGS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (7, 1, 128)]
LENS = [1, 15, 16, 17, 100, 333, 700]


def make_case(nh, nkv, hd, lens, kv, dtype, q_lens=None, bs=BS, seed=0, odd_scales=False):
    g = torch.Generator().manual_seed(seed + nh + hd)
    q_lens = q_lens or [1] * len(lens)
    nbs = [max(0, -(-L // bs)) for L in lens]
    nb = sum(nbs) + 5
    (k, ks), (v, vs) = [random_pool_fast(g, nb, bs, nkv, hd, kv) for _ in range(2)]
    if odd_scales:                                                              # any finite scale is a scale, zero too
        ks, vs = ks * (0.5 + torch.rand(ks.shape, generator=g)), vs * torch.exp2(torch.randint(-30, 3, vs.shape, generator=g).float()) * 1.3
        vs[0] = 0.0
    q = (torch.randn(sum(q_lens), nh, hd, generator=g) * 1.5).to(dtype)
    perm = torch.randperm(nb, generator=g).int()
    tables = torch.zeros(len(lens), max(max(nbs), 1), dtype=torch.int32)
    used = 0
    for i, n in enumerate(nbs):
        tables[i, :n] = perm[used:used + n]
        used += n
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32)
    return q, k, v, ks, vs, tables, torch.tensor(lens, dtype=torch.int32), cu


def random_pool_fast(g, nb, bs, nkv, hd, kv):
    x = torch.randn(nb, bs, nkv, hd, generator=g)
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=(1, 3)) / R.QMAX[kv])))
    return R.encode((x / s[:, None, :, None]).double(), kv).float().to(kv), s


def attend(case, decode, simple=False, **kw):
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    q, k, v, ks, vs, tables, lens, cu = [t.cuda() for t in case]
    return ragged_paged_attention(q, k, v, tables, lens, None if decode else cu, q.shape[-1] ** -0.5, k_scale=ks, v_scale=vs, simple=simple, **kw)


def check_attend(case, decode, simple=False, **kw):
    q, k, v, ks, vs, tables, lens, cu = case
    got = attend(case, decode, simple, **kw).cpu()
    kv, vv = R.values(k, ks), R.values(v, vs)
    sc = q.shape[-1] ** -0.5
    want = R.attend_fast(q, kv, vv, tables, lens, None if decode else cu, sc)
    tol = R.attend_tolerance(q, kv, vv, tables, lens, sc, want, q.dtype, None if (simple or q.dtype == torch.float32) else 11)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"max err {err.max().item():.3e}, worst err/tol {(err / tol).max().item():.2f}"


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", CONFIGS)
def test_decode(nh, nkv, hd, dtype, kv, simple):
    check_attend(make_case(nh, nkv, hd, LENS, kv, dtype), True, simple)


@pytest.mark.parametrize("nh,nkv,hd,bs", [(4, 4, 64, 16), (24, 2, 64, 16), (6, 3, 128, 16), (16, 1, 128, 32), (6, 2, 64, 64), (4, 2, 80, 16),
                                          (4, 2, 64, 8), (2, 1, 256, 16), (33, 3, 64, 16)])
@pytest.mark.parametrize("kv", KV8)
def test_decode_other_layouts(nh, nkv, hd, bs, kv):
    """Groups of 1, 2, 3, 11, 12 and 16 query heads, KV head counts that are no power of two, other block sizes and head dims."""
    check_attend(make_case(nh, nkv, hd, LENS, kv, torch.bfloat16, bs=bs), True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("lens", [[8192, 3, 4097, 16, 1, 777, 2048, 33, 5000, 64, 129, 6001], [20011], [9, 70000]])
def test_decode_long_rows_split(nh, nkv, hd, lens, dtype):
    """Rows over many CTAs next to short ones; twice on one workspace (its counters must be back at zero), bitwise equal."""
    from nanoserve_b200.kernels.paged_attention import AttnWorkspace
    case = make_case(nh, nkv, hd, lens, torch.int8, dtype, seed=1)
    ws = AttnWorkspace(64, 64, nh, hd)
    check_attend(case, True, workspace=ws)
    a, b = attend(case, True, workspace=ws), attend(case, True, workspace=ws)
    assert torch.equal(a, b)


def test_decode_many_short_rows():
    g = torch.Generator().manual_seed(7)
    lens = torch.randint(1, 200, (300,), generator=g).tolist()
    check_attend(make_case(14, 2, 64, lens, torch.int8, torch.bfloat16, seed=2), True)


@pytest.mark.parametrize("simple", [True, False])
def test_decode_rows_without_keys_are_zero(simple):
    case = list(make_case(14, 2, 64, [5, 1, 40], torch.int8, torch.bfloat16))
    case[6] = torch.tensor([0, 1, -3], dtype=torch.int32)
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    q, k, v, ks, vs, tables, lens, _ = [t.cuda() for t in case]
    out = ragged_paged_attention(q, k, v, tables, lens, None, 0.125, k_scale=ks, v_scale=vs, simple=simple)
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all()) and bool((out[1] != 0).any())


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("kv", KV8)
def test_odd_scales(kv, simple):
    """Scales that are no power of two, far apart, and zero."""
    check_attend(make_case(12, 2, 128, LENS, kv, torch.float32, odd_scales=True), True, simple)
    check_attend(make_case(14, 2, 64, LENS, kv, torch.bfloat16, odd_scales=True), True, simple)


MIXED = [([40, 52, 301, 17], [40, 22, 1, 1]), ([700, 16, 1, 512, 2048 + 512, 33], [1, 16, 1, 512, 512, 2]), ([5, 1, 1], [5, 1, 1]),
         ([130, 64, 65, 63, 200], [130, 64, 65, 63, 3]), ([100, 300], [0, 7])]


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("case", range(len(MIXED)))
@pytest.mark.parametrize("nh,nkv,hd,dtype", [(14, 2, 64, torch.bfloat16), (12, 2, 128, torch.bfloat16), (16, 2, 128, torch.bfloat16),
                                             (3, 3, 64, torch.bfloat16), (12, 2, 128, torch.float32), (24, 2, 64, torch.bfloat16)])
def test_mixed(nh, nkv, hd, dtype, case, kv, simple):
    lens, q_lens = MIXED[case]
    check_attend(make_case(nh, nkv, hd, lens, kv, dtype, q_lens), False, simple)


@pytest.mark.parametrize("kv", KV8)
def test_mixed_odd_scales(kv):
    lens, q_lens = MIXED[1]
    check_attend(make_case(14, 2, 64, lens, kv, torch.bfloat16, q_lens, odd_scales=True), False)
    check_attend(make_case(28, 4, 128, lens, kv, torch.bfloat16, q_lens, odd_scales=True), False)


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("kv", KV8)
def test_bad_block_ids_and_short_tables_are_absent_keys(kv, simple):
    """Ids outside the pool and lengths past the table's width: those keys do not exist; nothing is read there."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    case = list(make_case(4, 2, 64, [100, 60, 90, 40], kv, torch.bfloat16, [1, 20, 3, 1]))
    q, k, v, ks, vs, tables, lens, cu = case
    tables[0, 2], tables[0, 4], tables[1, 1], tables[3, 0], tables[3, 1], tables[3, 2] = -1, 2 ** 31 - 1, k.shape[0], -7, 99999, -1
    lens = torch.tensor([100, 60, 10 ** 6, 40], dtype=torch.int32)
    want = R.attend(q, R.values(k, ks), R.values(v, vs), tables, lens, cu, 0.125, BS)
    got = ragged_paged_attention(*[t.cuda() for t in (q, k, v, tables, lens, cu)], 0.125, k_scale=ks.cuda(), v_scale=vs.cuda(), simple=simple)
    tol = R.attend_tolerance(q, R.values(k, ks), R.values(v, vs), tables, torch.tensor([112]), 0.125, want, torch.bfloat16, 11)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert bool((got[-1] == 0).all())


@pytest.mark.parametrize("simple", [True, False])
def test_masked_places_may_hold_anything(simple):
    """NaN codes behind a sequence's last token, NaN scales and NaN codes in blocks no sequence owns, and rows of `out` behind
    the last sequence."""
    q, k, v, ks, vs, tables, lens, cu = make_case(14, 2, 64, [37, 61, 5], torch.float8_e4m3fn, torch.bfloat16, [1, 30, 1])
    nan = torch.full((1,), float("nan")).to(torch.float8_e4m3fn)
    kv, vv = R.values(k, ks), R.values(v, vs)
    for s, L in enumerate(lens.tolist()):
        b = tables[s, (L - 1) // BS]
        k[b, L % BS:], v[b, L % BS:] = nan, nan
    used = {int(tables[s, j]) for s, L in enumerate(lens.tolist()) for j in range(-(-L // BS))}
    for b in set(range(k.shape[0])) - used:
        k[b], v[b], ks[b], vs[b] = nan, nan, float("nan"), float("nan")
    qq = torch.cat((q, q[:6]))
    out = torch.full_like(qq, 7.0).cuda()
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    ragged_paged_attention(qq.cuda(), k.cuda(), v.cuda(), tables.cuda(), lens.cuda(), cu.cuda(), 0.125, k_scale=ks.cuda(), v_scale=vs.cuda(),
                           out=out, simple=simple)
    want = R.attend_fast(q, kv, vv, tables, lens, cu, 0.125)
    tol = R.attend_tolerance(q, kv, vv, tables, lens, 0.125, want, torch.bfloat16, 11)
    assert bool(((out.cpu()[:q.shape[0]].double() - want).abs() <= tol).all())
    assert bool((out[q.shape[0]:] == 7.0).all())


@pytest.mark.parametrize("simple", [True, False])
def test_nan_is_not_swallowed(simple):
    """A NaN in a query, and a NaN scale of a block that a sequence sees, reach the output; other rows are untouched."""
    case = make_case(14, 2, 64, [40, 40, 40, 90], torch.int8, torch.bfloat16, [1, 1, 1, 20])
    q, k, v, ks, vs, tables, lens, cu = case
    clean = attend(case, False, simple)
    q[1, 3, 5] = float("nan")
    vs[tables[2, 1]] = float("nan")
    ks[tables[3, 0], 1] = float("nan")
    out = attend(case, False, simple)
    assert bool(out[1, 3].isnan().all()) and bool(out[2].isnan().all()) and bool(out[3:, 7:].isnan().all())
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, 4:], clean[1, 4:]) and torch.equal(out[3:, :7], clean[3:, :7])


def test_strided_pools_queries_and_table_rows():
    """Pools with heads outside positions, a layer slice of a larger allocation, strided q and out rows, table_rows."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    q, k, v, ks, vs, tables, lens, cu = make_case(14, 2, 64, [100, 33, 64], torch.int8, torch.bfloat16, [1, 20, 64])
    kv, vv = R.values(k, ks), R.values(v, vs)
    perm = lambda t: t.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    ksd = torch.stack((ks, vs)).permute(0, 2, 1).contiguous().permute(0, 2, 1).cuda()
    rows = torch.tensor([2, 0, 1], dtype=torch.int32)
    shuffled = torch.zeros(3, tables.shape[1] + 3, dtype=torch.int32)
    for s in range(3):
        shuffled[rows[s], :tables.shape[1]] = tables[s]
    wide = torch.zeros(q.shape[0], q.shape[1] * 64 + 16, dtype=q.dtype)
    wide[:, :q.shape[1] * 64] = q.view(q.shape[0], -1)
    qs = wide.cuda()[:, :q.shape[1] * 64].unflatten(1, (q.shape[1], 64))
    ow = torch.zeros_like(wide).cuda()
    out = ow[:, :q.shape[1] * 64].unflatten(1, (q.shape[1], 64))
    ragged_paged_attention(qs, perm(k), perm(v), shuffled.cuda(), lens.cuda(), cu.cuda(), 0.125, table_rows=rows.cuda(), out=out,
                           k_scale=ksd[0], v_scale=ksd[1])
    want = R.attend_fast(q, kv, vv, tables, lens, cu, 0.125)
    tol = R.attend_tolerance(q, kv, vv, tables, lens, 0.125, want, torch.bfloat16, 11)
    assert bool(((out.cpu().double() - want).abs() <= tol).all()) and bool((ow[:, q.shape[1] * 64:] == 0).all())


# ------------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("kv", KV8)
def test_append_then_attend_over_steps(kv):
    """A prefill chunk, a second chunk on top and decode steps, as an engine makes them: tables, append, attention, with both
    pools followed by the plain forms."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    from nanoserve_b200.kernels.rotary import rope_append
    g = torch.Generator().manual_seed(11)
    nh, nkv, hd, nb = 14, 2, 64, 12
    tables = torch.randperm(nb, generator=g).int().view(2, 6)
    kc, vc = [torch.zeros(nb, BS, nkv, hd).to(kv).cuda() for _ in range(2)]
    ks, vs = [torch.zeros(nb, nkv).cuda() for _ in range(2)]
    ref = [(torch.zeros(nb, BS, nkv, hd).to(kv), torch.zeros(nb, nkv)) for _ in range(2)]
    have = [0, 0]
    for news in ([21, 9], [10, 1], [1, 1], [1, 1], [3, 1]):
        N = sum(news)
        pos = torch.cat([torch.arange(c, c + t) for c, t in zip(have, news)])
        slots = torch.cat([tables[s, torch.arange(c, c + t) // BS].long() * BS + torch.arange(c, c + t) % BS
                           for s, (c, t) in enumerate(zip(have, news))])
        have = [c + t for c, t in zip(have, news)]
        lens, cu = torch.tensor(have, dtype=torch.int32), torch.tensor([0, news[0], N], dtype=torch.int32)
        qkv = torch.randn(N, (nh + 2 * nkv) * hd, generator=g).bfloat16()
        cos, sin = tables_for(pos, hd)
        q, _, _ = rope_append(qkv.cuda(), cos, sin, nh, nkv, hd, kc, vc, slots.cuda(), k_scale=ks, v_scale=vs)
        out = ragged_paged_attention(q, kc, vc, tables.cuda(), lens.cuda(), cu.cuda(), 0.125, k_scale=ks, v_scale=vs)
        x = qkv.double().view(N, nh + 2 * nkv, hd)
        rot = R.rotate(x[:, :nh + nkv], cos.cpu(), sin.cpu(), False)
        for i, vals in enumerate((rot[:, nh:], x[:, nh + nkv:])):
            c, s = R.append(*ref[i], vals, slots.tolist())
            ref[i] = (c.float().to(kv), s.float())
        assert torch.equal(kc.cpu().float(), ref[0][0].float()) and torch.equal(vs.cpu(), ref[1][1])
        kvv, vvv = R.values(*ref[0]), R.values(*ref[1])
        want = R.attend_fast(rot[:, :nh].bfloat16(), kvv, vvv, tables, lens, cu, 0.125)
        tol = R.attend_tolerance(q.cpu(), kvv, vvv, tables, lens, 0.125, want, torch.bfloat16, 11)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())


def test_captured_and_replayed_with_new_lengths():
    """One graph over tables, append and attention (with and without a workspace of its own), replayed as the context grows;
    a second graph on another stream beside it."""
    from nanoserve_b200.kernels.paged_attention import paged_attention_decode
    from nanoserve_b200.kernels.rotary import rope_append, rope_tables, rotary_frequencies
    g = torch.Generator().manual_seed(12)
    nh, nkv, hd, B, nb = 14, 2, 64, 5, 40
    inv = rotary_frequencies(hd, 1e6)[0].cuda()

    def world():
        d = dict(tables=torch.randperm(nb, generator=g).int().view(B, 8).cuda(), lens=torch.ones(B, dtype=torch.int32).cuda(),
                 pos=torch.zeros(B, dtype=torch.int64).cuda(), slots=torch.zeros(B, dtype=torch.int64).cuda(),
                 qkv=torch.zeros(B, (nh + 2 * nkv) * hd, dtype=torch.bfloat16).cuda(),
                 k=torch.zeros(nb, BS, nkv, hd, dtype=torch.int8).cuda(), v=torch.zeros(nb, BS, nkv, hd, dtype=torch.int8).cuda(),
                 ks=torch.zeros(nb, nkv).cuda(), vs=torch.zeros(nb, nkv).cuda())

        def step():
            cos, sin = rope_tables(d["pos"], inv)
            q, _, _ = rope_append(d["qkv"], cos, sin, nh, nkv, hd, d["k"], d["v"], d["slots"], k_scale=d["ks"], v_scale=d["vs"])
            return q, paged_attention_decode(q, d["k"], d["v"], d["tables"], d["lens"], 0.125, k_scale=d["ks"], v_scale=d["vs"])
        return d, step

    worlds = [world(), world()]
    graphs, outs = [], []
    for d, step in worlds:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        for t in (d["k"], d["v"], d["ks"], d["vs"]):
            t.zero_()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step())
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in worlds]
    for n in range(40):
        inputs = [torch.randn(B, (nh + 2 * nkv) * hd, generator=g).bfloat16() for _ in worlds]
        for (d, _), x in zip(worlds, inputs):
            d["qkv"].copy_(x)
            d["pos"].fill_(n)
            d["lens"].fill_(n + 1)
            d["slots"].copy_(d["tables"][:, n // BS].long() * BS + n % BS)
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        if n in (0, 15, 16, 39):
            for (d, _), (q, o) in zip(worlds, outs):
                kv, vv = R.values(d["k"].cpu(), d["ks"].cpu()), R.values(d["v"].cpu(), d["vs"].cpu())
                want = R.attend_fast(q.cpu(), kv, vv, d["tables"].cpu(), d["lens"].cpu(), None, 0.125)
                tol = R.attend_tolerance(q.cpu(), kv, vv, d["tables"].cpu(), d["lens"].cpu(), 0.125, want, torch.bfloat16, 11)
                assert bool(((o.cpu().double() - want).abs() <= tol).all())


def test_two_streams_at_once():
    """Calls without a workspace on two streams do not share one."""
    cases = [make_case(14, 2, 64, [6000, 40, 3000], torch.int8, torch.bfloat16, seed=s) for s in (3, 4)]
    want = [attend(c, True) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    dev = [[t.cuda() for t in c] for c in cases]
    torch.cuda.synchronize()
    from nanoserve_b200.kernels.paged_attention import paged_attention_decode
    for _ in range(20):
        outs = []
        for st, (q, k, v, ks, vs, tables, lens, _) in zip(streams, dev):
            with torch.cuda.stream(st):
                outs.append(paged_attention_decode(q, k, v, tables, lens, 0.125, k_scale=ks, v_scale=vs))
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_empty_calls():
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    from nanoserve_b200.kernels.rotary import rope_append
    k = torch.zeros(2, BS, 2, 64, dtype=torch.int8).cuda()
    s = torch.zeros(2, 2).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    out = ragged_paged_attention(torch.zeros(0, 14, 64).bfloat16().cuda(), k, k, torch.zeros(0, 1, **i32), torch.zeros(0, **i32), None, 0.125,
                                 k_scale=s, v_scale=s)
    assert out.shape == (0, 14, 64)
    c = torch.zeros(0, 32).cuda()
    q, _, _ = rope_append(torch.zeros(0, 18 * 64).bfloat16().cuda(), c, c, 14, 2, 64, k, k.clone(), torch.zeros(0, dtype=torch.int64).cuda(),
                          k_scale=s, v_scale=s.clone())
    assert q.shape == (0, 14, 64)
