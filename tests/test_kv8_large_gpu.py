"""Appends of more than 256 tokens to 8-bit pools: the kernel that finds a block's tokens by looking through all slots."""
import pytest
import torch

from tests import kv8_reference as R
from tests.test_kv8_gpu import KV8, check_append, random_pool, tables_for

pytestmark = pytest.mark.gpu

# head dims with and without the paired fast path, block sizes 1 .. 64, part of the head, both pair layouts, no rotation
LAYOUTS = [(4, 2, 64, 64, 16, False), (2, 2, 128, 128, 16, False), (3, 1, 128, 128, 32, False), (2, 1, 64, 32, 16, True), (2, 1, 36, 20, 8, False),
           (2, 2, 64, 64, 64, False), (1, 1, 64, 0, 16, False), (2, 1, 64, 64, 1, False)]


def scattered(g, nb, bs, N, kind):
    if kind == "dups":                  # few slots, each named by many tokens of many chunks
        s = torch.randint(0, max(nb * bs // 8, 1), (N,), generator=g)
        s[50:90] = 5
        return s
    if kind == "own":                   # a block per token, as decode rows have
        s = torch.randperm(nb, generator=g)[:N] * bs + torch.randint(0, bs, (N,), generator=g)
        return s
    s = torch.arange(N) + 3             # a chunk that starts inside a block, then strays
    s[N - 9:] = torch.tensor([-1, nb * bs, 2 ** 40, -(2 ** 40), 0, nb * bs - 1, 1, 2, -5])
    return s


@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("kind", ["dups", "own", "chunk"])
@pytest.mark.parametrize("nh,nkv,hd,rot,bs,interleaved", LAYOUTS)
def test_large_append_is_the_definition(nh, nkv, hd, rot, bs, interleaved, kind, kv):
    g = torch.Generator().manual_seed(hd + rot + bs)
    N = 301
    nb = max(310, 40) if bs <= 16 or kind == "own" else 12
    slots = scattered(g, nb, bs, N, kind)
    qkv = (torch.randn(N, (nh + 2 * nkv) * hd, generator=g) * torch.exp2(torch.randint(-3, 4, (N, 1), generator=g).float())).bfloat16()
    cos, sin = tables_for(torch.arange(N), rot) if rot else (torch.empty(N, 0).cuda(),) * 2
    pools = [random_pool(g, nb, bs, nkv, hd, kv, s) for s in (0.1, 1.3)]
    check_append(qkv, cos, sin, nh, nkv, hd, pools, slots, interleaved)


@pytest.mark.parametrize("kv", KV8)
@pytest.mark.parametrize("hd", [64, 80])
def test_large_append_of_values_that_are_not_finite(hd, kv):
    """Infinities and NaN in a few tokens, pools whose scales are NaN, zero or no power of two."""
    g = torch.Generator().manual_seed(hd)
    nkv, nb, N = 2, 40, 400
    slots = torch.randperm(nb * 16, generator=g)[:N]
    qkv = torch.randn(N, 3 * nkv * hd, generator=g)
    x = qkv.view(N, 3 * nkv, hd)
    x[3, nkv, 1], x[200, nkv + 1, 0], x[333, 2 * nkv, 7] = float("nan"), float("inf"), float("-inf")
    pools = [random_pool(g, nb, 16, nkv, hd, kv) for _ in range(2)]
    pools[0][1][1], pools[0][1][2], pools[1][1][3], pools[1][1][4] = float("nan"), 0.0, 0.037, float("nan")
    cos, sin = torch.empty(N, 0).cuda(), torch.empty(N, 0).cuda()
    check_append(qkv, cos, sin, nkv, nkv, hd, pools, slots)


@pytest.mark.parametrize("interleaved", [False, True])
def test_large_append_with_dense_copies_and_strided_rows(interleaved):
    """dense_kv beside an 8-bit pool, rows of qkv inside a wider buffer, pools with heads outside positions: the same codes, and
    dense K and V as of a call without a pool."""
    from nanoserve_b200.kernels.rotary import rope_append
    g = torch.Generator().manual_seed(3)
    nh, nkv, hd, nb, N = 4, 2, 64, 30, 290
    width = (nh + 2 * nkv) * hd
    wide = torch.randn(N, width + 64, generator=g).bfloat16().cuda()
    qkv = wide[:, :width]
    cos, sin = tables_for(torch.arange(N) + 1000, hd)
    slots = torch.randperm(nb * 16, generator=g)[:N].cuda()
    pools = [random_pool(g, nb, 16, nkv, hd, torch.int8) for _ in range(2)]
    plain = [t.cuda() for p in pools for t in p]
    other = [t.clone() if t.dim() == 2 else t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in plain]
    q0, _, _ = rope_append(qkv.contiguous(), cos, sin, nh, nkv, hd, plain[0], plain[2], slots, k_scale=plain[1], v_scale=plain[3],
                           interleaved=interleaved)
    q1, k1, v1 = rope_append(qkv, cos, sin, nh, nkv, hd, other[0], other[2], slots, k_scale=other[1], v_scale=other[3], interleaved=interleaved,
                             dense_kv=True)
    q2, k2, v2 = rope_append(qkv, cos, sin, nh, nkv, hd, dense_kv=True, interleaved=interleaved)
    assert torch.equal(q0, q1) and torch.equal(q0, q2) and torch.equal(k1, k2) and torch.equal(v1, v2)
    for a, b in zip(plain, other):
        assert torch.equal(a, b)
    rot = R.rotate(qkv.cpu().double().view(N, nh + 2 * nkv, hd)[:, :nh + nkv], cos.cpu(), sin.cpu(), interleaved)
    assert torch.equal(k2.cpu(), rot[:, nh:].bfloat16()) and torch.equal(v2.cpu().view(N, -1), qkv.cpu()[:, (nh + nkv) * hd:])


def test_appends_of_one_stream_follow_each_other():
    """Large and small steps into the same blocks, back to back, replayed from a graph: each finds what the one before left."""
    from nanoserve_b200.kernels.rotary import kv_values, rope_append
    g = torch.Generator().manual_seed(9)
    nh, nkv, hd, nb = 2, 1, 64, 24
    steps = []
    for N in (300, 40, 280, 1, 310):
        cos, sin = tables_for(torch.arange(N), hd)
        steps.append((torch.randn(N, 4 * hd, generator=g).bfloat16().cuda() * (N % 7 + 1), cos, sin, torch.randperm(nb * 16, generator=g)[:N].cuda()))
    start = [t.cuda() for p in [random_pool(g, nb, 16, nkv, hd, torch.float8_e4m3fn) for _ in range(2)] for t in p]
    want = [[t.cpu() for t in start]]
    for qkv, cos, sin, slots in steps:
        x = qkv.cpu().double().view(-1, 4, hd)
        rot = R.rotate(x[:, :3], cos.cpu(), sin.cpu(), False)
        last, new = want[-1], []
        for (pool, scale), vals in (((last[0], last[1]), rot[:, 2:]), ((last[2], last[3]), x[:, 3:])):
            codes, sc = R.append(pool, scale, vals, slots.tolist())
            new += [codes.float().to(torch.float8_e4m3fn), sc.float()]
        want.append(new)
    live = [t.clone() for t in start]

    def run():
        for qkv, cos, sin, slots in steps:
            rope_append(qkv, cos, sin, nh, nkv, hd, live[0], live[2], slots, k_scale=live[1], v_scale=live[3])

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        for t, s in zip(live, start):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip(live, want[-1]):
            assert torch.equal(got.cpu().float(), w.float())
    assert torch.equal(kv_values(live[0], live[1]).cpu(), R.values(want[-1][0], want[-1][1]).float())
