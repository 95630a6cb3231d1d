"""Prefill chunks over 8-bit pools that are split over their keys: few chunks, many keys (long prompts served alone)."""
import pytest
import torch

from tests import kv8_reference as R
from tests.test_kv8_gpu import BS, KV8, attend, check_attend, make_case

pytestmark = pytest.mark.gpu

# (lens, new tokens): an item is 32 tokens of a KV head and is split from 8 tiles of 64 keys on. One 16-token tile; odd tails; a
# decode row and short items beside a long one; parts that end inside a block's tile; all keys new.
SPLIT = [([1000], [16]), ([700], [100]), ([513, 1, 2049], [33, 1, 470]), ([2600, 37], [512, 5]), ([449, 448, 512], [17, 17, 64]), ([640], [640])]


@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("case", range(len(SPLIT)))
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (28, 4, 128), (3, 3, 64), (24, 2, 128)])
def test_split_chunks(nh, nkv, hd, case, kv):
    lens, q_lens = SPLIT[case]
    check_attend(make_case(nh, nkv, hd, lens, kv, torch.bfloat16, q_lens), False)


@pytest.mark.parametrize("kv", KV8)
def test_split_chunks_odd_scales_and_block_sizes(kv):
    lens, q_lens = SPLIT[2]
    check_attend(make_case(14, 2, 64, lens, kv, torch.bfloat16, q_lens, odd_scales=True), False)
    check_attend(make_case(28, 4, 128, lens, kv, torch.bfloat16, q_lens, odd_scales=True), False)
    check_attend(make_case(14, 2, 64, lens, kv, torch.bfloat16, q_lens, bs=64), False)
    check_attend(make_case(12, 2, 128, lens, kv, torch.bfloat16, q_lens, bs=32), False)


@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (7, 1, 128)])
def test_split_parts_without_a_key(nh, nkv, hd):
    """Whole parts of a chunk's keys absent (block ids outside the pool), then all of them: other rows and parts do not notice."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    case = list(make_case(nh, nkv, hd, [800, 520], torch.int8, torch.bfloat16, [20, 3]))
    q, k, v, ks, vs, tables, lens, cu = case
    kv, vv = R.values(k, ks), R.values(v, vs)
    for rows in ([slice(0, 14)], [slice(12, 37)], [slice(0, 12), slice(25, 51)], [slice(0, 51)]):
        t = tables.clone()
        for r in rows:
            t[0, r] = -1
        want = R.attend(q, kv, vv, t, lens, cu, hd ** -0.5, BS)
        got = ragged_paged_attention(*[x.cuda() for x in (q, k, v, t, lens, cu)], hd ** -0.5, k_scale=ks.cuda(), v_scale=vs.cuda())
        tol = R.attend_tolerance(q, kv, vv, t, lens, hd ** -0.5, want, torch.bfloat16, 11)
        assert bool(((got.cpu().double() - want).abs() <= tol).all())


def test_split_nan_reaches_the_rows_that_see_it_and_no_other():
    """A NaN scale in a block of one part; NaN codes (K and V) at a position that only the later tokens of the chunk see."""
    case = make_case(14, 2, 64, [1024], torch.float8_e4m3fn, torch.bfloat16, [64])
    q, k, v, ks, vs, tables, lens, cu = case
    clean = attend(case, False)
    nan = torch.full((1,), float("nan")).to(torch.float8_e4m3fn)
    late = tables[0, 1000 // BS]
    for pool in (k, v):                                        # token 1000: rows 40 .. 63 of the chunk see it
        keep = pool[late, 1000 % BS, 1].clone()
        pool[late, 1000 % BS, 1] = nan
        out = attend(case, False)
        assert torch.equal(out[:40], clean[:40]) and torch.equal(out[:, :7], clean[:, :7]) and bool(out[40:, 7:].isnan().all())
        pool[late, 1000 % BS, 1] = keep
    for scale in (ks, vs):
        keep = scale[tables[0, 5], 0].clone()
        scale[tables[0, 5], 0] = float("nan")
        out = attend(case, False)
        assert bool(out[:, :7].isnan().all()) and torch.equal(out[:, 7:], clean[:, 7:])
        scale[tables[0, 5], 0] = keep
    assert torch.equal(attend(case, False), clean)


def test_split_captured_then_replayed_with_other_lengths():
    """One captured launch serves lengths on both sides of the split: the device decides."""
    from nanoserve_b200.kernels.paged_attention import AttnWorkspace, ragged_paged_attention
    q, k, v, ks, vs, tables, lens, cu = make_case(14, 2, 64, [1500], torch.int8, torch.bfloat16, [48])
    kv, vv = R.values(k, ks), R.values(v, vs)
    d = [t.cuda() for t in (q, k, v, tables, lens, cu)]
    ksd, vsd = ks.cuda(), vs.cuda()
    ws = AttnWorkspace(64, 4, 14, 64)
    out = torch.zeros_like(d[0])

    def call():
        ws.plan(d[4], d[5], 1, BS)
        ragged_paged_attention(*d, 0.125, workspace=ws, planned=True, out=out, k_scale=ksd, v_scale=vsd)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n in (1500, 48, 447, 448, 449, 513, 1280):
        d[4].fill_(n)
        graph.replay()
        want = R.attend_fast(q, kv, vv, tables, torch.tensor([n]), cu, 0.125)
        tol = R.attend_tolerance(q, kv, vv, tables, torch.tensor([n]), 0.125, want, torch.bfloat16, 11)
        assert bool(((out.cpu().double() - want).abs() <= tol).all()), n


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("lens,q_lens", [([5, 30], [40, 33]), ([600, 3, 1], [700, 16, 1])])
def test_fewer_keys_than_tokens(lens, q_lens, simple):
    """A chunk longer than its sequence: the first tokens see nothing and get zeros, the others what is left of the keys."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    q, k, v, ks, vs, tables, lens, cu = make_case(4, 2, 64, lens, torch.int8, torch.bfloat16, q_lens)
    kv, vv = R.values(k, ks), R.values(v, vs)
    want = R.attend_fast(q, kv, vv, tables, lens, cu, 0.125)
    got = ragged_paged_attention(*[x.cuda() for x in (q, k, v, tables, lens, cu)], 0.125, k_scale=ks.cuda(), v_scale=vs.cuda(), simple=simple)
    tol = R.attend_tolerance(q, kv, vv, tables, lens, 0.125, want, torch.bfloat16, None if simple else 11)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())
    assert bool((got[:q_lens[0] - int(lens[0])] == 0).all())


@pytest.mark.parametrize("simple", [True, False])
@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("lens,q_lens", [([300, 40, 9], [1, 1, 1]), ([700, 50], [90, 17])])
def test_scales_of_the_scores_that_are_not_positive(lens, q_lens, scale, simple):
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    q, k, v, ks, vs, tables, lens, cu = make_case(14, 2, 64, lens, torch.float8_e4m3fn, torch.bfloat16, q_lens)
    kv, vv = R.values(k, ks), R.values(v, vs)
    want = R.attend_fast(q, kv, vv, tables, lens, cu, scale)
    got = ragged_paged_attention(*[x.cuda() for x in (q, k, v, tables, lens, cu)], scale, k_scale=ks.cuda(), v_scale=vs.cuda(), simple=simple)
    tol = R.attend_tolerance(q, kv, vv, tables, lens, abs(scale), want, torch.bfloat16, None if simple else 11)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


def test_calls_on_another_stream_than_the_default():
    """Append and attention on a side stream, the plan included, while the default stream is busy with something else."""
    from nanoserve_b200.kernels.paged_attention import ragged_paged_attention
    case = make_case(14, 2, 64, [700, 1, 90], torch.int8, torch.bfloat16, [100, 1, 8])
    want = attend(case, False)
    q, k, v, ks, vs, tables, lens, cu = [t.cuda() for t in case]
    torch.cuda.synchronize()
    noise = torch.randn(2048, 2048, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(5):
        noise = (noise @ noise).clamp(-1, 1)
        with torch.cuda.stream(side):
            got = ragged_paged_attention(q, k, v, tables, lens, cu, 0.125, k_scale=ks, v_scale=vs)
        side.synchronize()
        assert torch.equal(got, want)
