"""Expert routing, 8-bit integer products and draft verification on the GPU
against their definitions in float64.

Tolerances count roundings.  U = 2^-24 is half a step of fp32.  Routing weights
are 64 bits until they are stored: half a step of fp32.  Sums of integer products
are exact; a result is their conversion to fp32, two products with scales and one
sum with the bias, each half a step of its result, and half a step of its type as
it is stored.  Ids and codes are equal.
"""
import math

import numpy as np
import pytest
import torch

from vibeblade_amd import ggml
from vibeblade_amd.gpu import HipBackend
from vibeblade_amd.int8 import K_MAX, Int8QTensor, int8_gemm, quantize_tokens
from vibeblade_amd.moe import ExpertRouter, MoEExpertSet, moe_ffn_silu
from vibeblade_amd.moe_executor import HotColdExecutor
from vibeblade_amd.moe_profiler import HotColdMap
from vibeblade_amd.tensor import (QTensor, block_norm, gemm, moe_grouped_ffn, moe_route, route_experts, token_logprobs,
                                  verify_draft)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = math.inf


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    yield


def normal(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def uniform(seed, *shape):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed))


def half_step(want, dtype):
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def close(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = ((got - want).abs() - tol)[~torch.isnan(want)]
    assert off.numel() == 0 or off.max() <= 0, f"{off.max():.3e} over the tolerance"


# ---- route_experts ------------------------------------------------------------------

def route64(z, topk, scores="softmax", bias=None, groups=1, groups_kept=None, group_score="max", renorm=True, scale=1.0):
    """One token and one expert at a time."""
    z = z.double().numpy()
    b = np.zeros(z.shape[1]) if bias is None else bias.double().numpy()
    kept, size = groups if groups_kept is None else groups_kept, z.shape[1] // groups
    ids = np.full((z.shape[0], topk), -1, dtype=np.int32)
    ws = np.zeros((z.shape[0], topk))
    for t, row in enumerate(z):
        with np.errstate(all="ignore"):
            if scores == "softmax":
                e = np.exp(row - row.max())
                s = np.zeros_like(row) if row.max() == -INF else e / e.sum()
            else:
                s = 1 / (1 + np.exp(-row))
        value = s + b
        choice = row if bias is None else value
        if np.isnan(choice).any() or np.isnan(s).any():
            ws[t] = math.nan
            continue
        open_ = (row > -INF) & (b > -INF)
        if kept < groups:
            ranks = []
            for g in range(groups):
                of = np.arange(g * size, (g + 1) * size)
                of = of[open_[of]]
                if group_score == "max":
                    rank = max((choice[e] for e in of), default=-INF)
                else:
                    two = sorted((value[e] for e in of), reverse=True)[:2]
                    rank = sum(two) if two else -INF
                ranks.append((-rank, g))
            stay = {g for _, g in sorted(ranks)[:kept]}
            open_ &= np.array([e // size in stay for e in range(z.shape[1])])
        best = sorted((-choice[e], e) for e in range(z.shape[1]) if open_[e])[:topk]
        for j, (_, e) in enumerate(best):
            ids[t, j], ws[t, j] = e, s[e]
        if renorm:
            total = ws[t].sum()
            ws[t] = ws[t] / total if total > 0 else 0.0
    return torch.from_numpy(ids), torch.from_numpy(ws * scale)


def check_route(z, topk, bias=None, **kw):
    ids, w = route_experts(z.cuda(), topk, bias=None if bias is None else bias.cuda(), **kw)
    want_ids, want_w = route64(z, topk, bias=bias, **kw)
    assert ids.dtype == torch.int32 and w.dtype == F32
    assert torch.equal(ids.cpu(), want_ids)
    # 64-bit values to 2^-50 of each other, then one rounding
    close(w, want_w, half_step(want_w, F32) + 2.0 ** -50 * want_w.abs())


@pytest.mark.parametrize("experts,topk", [(1, 1), (2, 1), (2, 2), (7, 3), (60, 4), (64, 8), (65, 8), (128, 8), (129, 6),
                                          (160, 6), (256, 8), (257, 10), (384, 8), (511, 22), (512, 64)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [1, 5, 130])
def test_route_experts_sizes(experts, topk, scores, tokens):
    z = normal(experts + tokens, tokens, experts, scale=1.5)
    check_route(z, topk, scores=scores)
    check_route(z, topk, scores=scores, bias=0.1 * normal(9, experts), renorm=False, scale=2.5)


@pytest.mark.parametrize("groups,size,kept", [(2, 1, 1), (3, 5, 2), (4, 64, 2), (5, 13, 2), (6, 20, 1), (8, 20, 3), (8, 32, 4),
                                              (8, 64, 7), (16, 16, 5), (33, 15, 9), (64, 8, 32), (64, 1, 10), (4, 2, 4),
                                              (1, 100, 1)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_experts_groups(groups, size, kept, group_score, bias):
    experts, topk = groups * size, min(8, kept * size)
    z = normal(groups, 37, experts, scale=1.5)
    b = 0.1 * normal(4, experts) if bias else None
    for scores in ("softmax", "sigmoid"):
        check_route(z, topk, bias=b, scores=scores, groups=groups, groups_kept=kept, group_score=group_score)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 3)])
def test_route_experts_ties_go_to_the_lower_id(dtype, groups, kept):
    z = normal(3, 200, 160, scale=1.0).mul(2).round().div(2).to(dtype)  # a few values only
    for group_score in ("max", "top2"):
        check_route(z, 8, groups=groups, groups_kept=kept, group_score=group_score)
    check_route(z, 8, groups=groups, groups_kept=kept, bias=torch.zeros(160), scores="sigmoid")
    check_route(torch.zeros(3, 160, dtype=dtype), 8, groups=groups, groups_kept=kept)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (8, 2)])
@pytest.mark.parametrize("bias", [False, True])
def test_route_experts_masks(scores, groups, kept, bias):
    z = normal(11, 40, 64, scale=2.0)
    z[uniform(12, 40, 64) < 0.8] = -INF
    z[3], z[4], z[5], z[6] = -INF, -INF, torch.finfo(F32).min, -1e4
    z[4, 17] = 1.0
    b = 0.1 * normal(5, 64) if bias else None
    if bias:
        b[9] = b[33] = -INF
    for group_score in ("max", "top2"):
        for renorm in (True, False):
            check_route(z, 6, bias=b, scores=scores, groups=groups, groups_kept=kept, group_score=group_score, renorm=renorm)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_experts_nan_and_infinities(scores, bias):
    z = normal(13, 9, 100)
    z[1, 7] = math.nan
    z[3, 99] = INF
    z[5, 0], z[5, 3] = math.nan, -INF
    z[7, 50], z[7, 51] = 3e38, -3e38
    b = 0.1 * normal(5, 100) if bias else None
    check_route(z, 5, bias=b, scores=scores)
    check_route(z, 5, bias=b, scores=scores, groups=10, groups_kept=4, group_score="top2")
    if bias:
        b[20], b[21] = INF, -INF
        check_route(z, 5, bias=b, scores=scores)
        b[20] = math.nan
        check_route(z, 5, bias=b, scores=scores)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_route_experts_group_sums_past_fp32(scores, sign):
    """Two biases whose sum is no fp32 number: groups are told apart in 64 bits all the same."""
    z = normal(27, 20, 12)
    b = torch.tensor([3.0, 2.9, 0.0, 0.0, 3.3, 3.2, 0.0, 0.0, 3.1, 3.0, 0.0, 0.0]) * 1e38
    if sign < 0:
        b = -torch.tensor([3.3, 3.2, 3.35, 3.25, 3.0, 2.9, 3.1, 3.05, 3.2, 3.1, 3.3, 3.15]) * 1e38
    for kept, topk in ((1, 1), (1, 2), (2, 3)):
        check_route(z, topk, bias=b, scores=scores, groups=3, groups_kept=kept, group_score="top2")


def test_route_experts_scores_closer_than_fp32_are_told_apart():
    # sigmoid(z) + b of neighbours differ by 2^-30 or less: equal in fp32
    z = torch.zeros(64, 128)
    b = torch.zeros(128)
    for t in range(64):
        z[t, t + 3] = 2.0 ** -26 * (1 + t)
        z[t, 2 * t + 1 if 2 * t + 1 != t + 3 else 0] = 2.0 ** -27
    check_route(z, 3, bias=b, scores="sigmoid")
    check_route(z, 3, bias=b + 0.25, scores="softmax")


def test_route_experts_strides_and_no_tokens():
    wide = normal(17, 50, 300)
    for z in (wide[:, 5:133], wide[::3, 7:107], wide.T[:100], wide[7:8].expand(6, 300), wide[:1, :64]):
        ids, w = route_experts(z.cuda() if z.is_contiguous() else torch.empty_strided(
            z.shape, z.stride(), device="cuda").copy_(z) if 0 not in z.stride() else z[:1].cuda().expand(z.shape), 4)
        want_ids, want_w = route64(z, 4)
        assert torch.equal(ids.cpu(), want_ids)
        close(w, want_w, half_step(want_w, F32) + 2.0 ** -50 * want_w.abs())
    ids, w = route_experts(torch.empty(0, 8, device="cuda"), 2)
    assert ids.shape == w.shape == (0, 2)


def test_route_experts_many_tokens():
    z = normal(19, 5001, 256, scale=1.5)
    check_route(z, 8, bias=0.1 * normal(20, 256), scores="sigmoid", groups=8, groups_kept=4, group_score="top2", scale=2.5)


def test_route_experts_agrees_with_the_clamped_routing_inside_its_range():
    z = normal(23, 77, 64).cuda()
    (ids, w), (old_ids, old_w) = route_experts(z, 8), moe_route(z, 8)
    assert torch.equal(ids, old_ids)
    assert (w - old_w).abs().max() < 2e-6  # that one is fp32 throughout


def test_route_experts_refusals():
    z = torch.zeros(4, 64, device="cuda")
    for bad in (dict(topk=0), dict(topk=65), dict(topk=2, scores="relu"), dict(topk=2, group_score="mean"),
                dict(topk=2, groups=5), dict(topk=2, groups=8, groups_kept=0), dict(topk=9, groups=8, groups_kept=1),
                dict(topk=2, bias=torch.zeros(63, device="cuda")), dict(topk=2, bias=torch.zeros(64)),
                dict(topk=2, bias=torch.zeros(64, device="cuda", dtype=F16)), dict(topk=2, scale=INF)):
        with pytest.raises(ValueError):
            route_experts(z, **bad)
    for bad in (z[0], z.double(), torch.zeros(4, 513, device="cuda"), torch.zeros(4, 0, device="cuda")):
        with pytest.raises(ValueError):
            route_experts(bad, 1)


# ---- the experts of a given routing ------------------------------------------------------

def make_experts(n_exp, h, i, qtype=ggml.GGML_TYPE_Q4_K, seed=0):
    def some(s, r, c):
        return [QTensor.quantize(normal(seed + 1000 * s + e, r, c, scale=0.05), qtype, device="cuda") for e in range(n_exp)]
    return some(1, i, h), some(2, i, h), some(3, h, i)


def experts64(experts, x, ids, w):
    gates, ups, downs = ([q.dequantize().cpu().double() for q in qs] for qs in experts)
    y = torch.zeros(x.shape, dtype=torch.float64)
    for t in range(x.shape[0]):
        for e, we in zip(ids[t].tolist(), w[t].double().tolist()):
            if 0 <= e < len(gates):
                g, u = gates[e] @ x[t].double(), ups[e] @ x[t].double()
                y[t] += we * (downs[e] @ (g / (1 + torch.exp(-g)) * u))
    return y


def rel_l2(got, want):
    return float((got.cpu().double() - want).norm() / want.norm())


@pytest.mark.parametrize("qtype", [ggml.GGML_TYPE_Q4_K, ggml.GGML_TYPE_Q8_0, ggml.GGML_TYPE_F32])
@pytest.mark.parametrize("tokens,topk", [(1, 1), (1, 2), (9, 2), (33, 3), (70, 8)])
def test_experts_of_a_given_routing(qtype, tokens, topk):
    experts = make_experts(8, 256, 512, qtype)
    x, z = normal(1, tokens, 256), normal(2, tokens, 8)
    routing = route_experts(z.cuda(), topk, scores="sigmoid", scale=1.5)
    y, ids, w = moe_grouped_ffn(*experts, x.cuda(), routing=routing)
    assert ids is not None and torch.equal(ids, routing[0]) and torch.equal(w, routing[1])
    # the products' own bound on the fp16 matrix path
    assert rel_l2(y, experts64(experts, x, ids.cpu(), w.cpu())) < 5e-3


def test_experts_of_a_given_routing_as_of_the_logits():
    """The same routing handed in: the same bits."""
    experts = make_experts(8, 256, 512)
    for tokens, topk in ((4, 2), (20, 2), (100, 2), (16, 4), (100, 8)):
        x, z = normal(1, tokens, 256).cuda(), normal(2, tokens, 8).cuda()
        y, ids, w = moe_grouped_ffn(*experts, x, z, topk)
        again, _, _ = moe_grouped_ffn(*experts, x, routing=(ids, w))
        assert torch.equal(y, again)


def test_experts_that_are_not_there_add_nothing():
    experts = make_experts(4, 256, 256)
    x = normal(3, 6, 256)
    for topk in (2, 3):
        ids = torch.full((6, topk), -1, dtype=torch.int32)
        ids[1, 0], ids[2], ids[3, 1], ids[4, 0] = 3, 2, 4, 1 << 30  # the same one twice; past the last
        w = uniform(4, 6, topk)
        w[0] = math.nan
        y, _, _ = moe_grouped_ffn(*experts, x.cuda(), routing=(ids.cuda(), w.cuda()))
        want = experts64(experts, x, ids, w.nan_to_num(0.0))
        assert not y[[0, 3, 4, 5]].any()
        assert rel_l2(y, want) < 5e-3


@pytest.mark.parametrize("n_exp,topk,tokens", [(70, 4, 5), (130, 12, 9), (3, 2, 1100), (2, 5, 4)])
def test_experts_past_the_limits_of_a_call(n_exp, topk, tokens):
    experts = make_experts(n_exp, 256, 256)
    x, z = normal(5, tokens, 256), normal(6, tokens, n_exp)
    if topk <= n_exp:
        ids, w = route_experts(z.cuda(), topk)
    else:
        ids = torch.randint(0, n_exp, (tokens, topk), dtype=torch.int32, device="cuda")
        w = uniform(7, tokens, topk).cuda()
    y, _, _ = moe_grouped_ffn(*experts, x.cuda(), routing=(ids, w))
    some = slice(0, tokens) if tokens < 100 else slice(tokens - 90, tokens)
    assert rel_l2(y[some], experts64(experts, x[some], ids[some].cpu(), w[some].cpu())) < 5e-3


def test_given_routing_refusals():
    experts = make_experts(2, 256, 256)
    x, ids, w = torch.zeros(3, 256, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    for bad in (dict(), dict(logits=torch.zeros(3, 2, device="cuda"), topk=1, routing=(ids, w)), dict(logits=w),
                dict(routing=(ids.long(), w)), dict(routing=(ids, w.half())), dict(routing=(ids[:2], w[:2])),
                dict(routing=(ids, w[:, :1])), dict(routing=(ids.cpu(), w)), dict(routing=(ids[:, :0], w[:, :0]))):
        with pytest.raises(ValueError):
            moe_grouped_ffn(*experts, x, **bad)
    with pytest.raises(ValueError):
        moe_grouped_ffn(*experts, torch.zeros(3, 512, device="cuda"), routing=(ids, w))


def test_router_with_options_in_the_layer_and_the_executor():
    rng = np.random.RandomState(0)
    h, inter, n_exp = 64, 96, 16
    gate, up, down = (rng.randn(n_exp, *s).astype(np.float32) * 0.1 for s in ((inter, h), (inter, h), (h, inter)))
    bias = rng.randn(n_exp).astype(np.float32) * 0.1
    options = dict(scores="sigmoid", bias=bias, groups=4, groups_kept=2, group_score="top2", scale=2.5)
    router = ExpertRouter(rng.randn(h, n_exp).astype(np.float32) * 0.1, 3, **options)
    x = rng.randn(7, h).astype(np.float32)
    experts = MoEExpertSet(gate, up, down)
    out, stats = moe_ffn_silu(x, router, experts)
    z = torch.from_numpy(router.predict(x))  # the logits that were routed
    ids, w = route64(z, 3, **{**options, "bias": torch.from_numpy(bias)})
    assert np.array_equal(stats["expert_indices"], ids.numpy())
    routed_ids, routed_w = router.route(x)
    assert np.array_equal(routed_ids, ids.numpy()) and np.allclose(routed_w, w.numpy(), rtol=1e-6)
    want = np.zeros_like(x, dtype=np.float64)
    for t in range(7):
        for e, we in zip(ids[t].tolist(), w[t].tolist()):
            g, u = gate[e].astype(np.float64) @ x[t], up[e].astype(np.float64) @ x[t]
            want[t] += we * (down[e].astype(np.float64) @ (g / (1 + np.exp(-g)) * u))
    assert np.linalg.norm(out - want) < 5e-3 * np.linalg.norm(want)
    ex = HotColdExecutor(HotColdMap({0: list(range(n_exp))}, {0: []}, 1, n_exp), {0: router}, {0: experts})
    again, stats = ex.dispatch(0, x)
    assert np.array_equal(again, out) and stats["gpu_hits"] == 21


# ---- 8-bit integer products -----------------------------------------------------------------

def scales64(x):
    """The rows' scales in fp32: the quotient in 64 bits, rounded once."""
    s = (x.double().abs().amax(1) / 127).float().clamp(min=2.0 ** -126)
    return torch.where(x.abs().amax(1) > 0, s, 0.0)


def codes64(x, s):
    return torch.where(s[:, None] > 0, (x.double() / s.double()[:, None]).round(), 0.0)


def codes_of(q):
    """The codes of a packed matrix, from its bytes."""
    tiles, blocks = (q.rows + 15) // 16, (q.k + 63) // 64
    b = q.data[:tiles * blocks * 1024].view(torch.int8).cpu().view(tiles, blocks, 4, 16, 16)  # tile, block, k / 16, row, k
    return b.permute(0, 3, 1, 2, 4).reshape(tiles * 16, blocks * 64)


@pytest.mark.parametrize("rows,k", [(1, 1), (1, 4096), (15, 63), (16, 64), (17, 65), (40, 1000), (5, 14336), (3, 20001)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_int8_quantize(rows, k, dtype):
    x = normal(rows + k, rows, k)
    x[uniform(1, rows, k) < 0.01] *= 20
    x = x.to(dtype)
    x[rows // 2] = 0
    q = quantize_tokens(x.cuda())
    s = scales64(x)
    assert torch.equal(q.scales.cpu(), s)
    all_codes = codes_of(q)
    assert torch.equal(all_codes[:rows, :k].double(), codes64(x, s))
    assert not all_codes[rows:].any() and not all_codes[:, k:].any()  # what the products read past the matrix
    assert torch.equal(q.dequantize().cpu(), all_codes[:rows, :k].float() * s[:, None])


def test_int8_quantize_ties_and_their_neighbours():
    # s = 1 (the row's largest is 127): halves are ties, and one step beside them are none
    half = torch.arange(-126, 126).float() + 0.5
    row = torch.cat([torch.tensor([127.0]), half, torch.nextafter(half, torch.tensor(INF)), torch.nextafter(half, torch.tensor(-INF))])
    x = torch.stack([row, row * 2.0 ** -120, row * 2.0 ** 100, row * 0.3, row * 1.7e-3, -row * 123.456])
    q = quantize_tokens(x.cuda())
    s = scales64(x)
    assert torch.equal(q.scales.cpu(), s)
    assert torch.equal(codes_of(q)[:6, :row.numel()].double(), codes64(x, s))


def test_int8_quantize_small_large_and_unbounded_rows():
    x = normal(3, 8, 200)
    x[0] *= 2.0 ** -149 / x[0].abs().max()  # nothing but the smallest subnormals and zeros
    x[1] *= 1e-40
    x[2] *= 1e-37
    x[3] *= 3e38 / x[3].abs().max()
    x[4, 7], x[5, 199], x[6, 0] = math.nan, INF, -INF
    q = quantize_tokens(x.cuda())
    s = scales64(x[[0, 1, 2, 3, 7]])
    assert torch.equal(q.scales.cpu()[[0, 1, 2, 3, 7]], s)
    assert torch.equal(codes_of(q)[[0, 1, 2, 3, 7], :200].double(), codes64(x[[0, 1, 2, 3, 7]], s))
    assert torch.isnan(q.scales.cpu()[4:7]).all() and not codes_of(q)[4:7].any()


def product64(qx, sx, qw, sw, bias, out_dtype):
    """(y, tolerance): sums exact; roundings as the module says."""
    p = (qx.double() @ qw.double().T) * sx.double()[:, None] * sw.double()
    y = p if bias is None else p + bias.double()
    tol = 3.01 * U * p.abs() + (0 if bias is None else U * y.abs())
    # an fp32 result is the last of these roundings
    return y, tol + (0 if out_dtype == F32 else half_step(y.abs() + tol, out_dtype))


def check_product(m, n, k, x_dtype=F32, out_dtype=F32, bias=False, packed=False, seed=0):
    qw = torch.randint(-128, 128, (n, k), generator=torch.Generator().manual_seed(seed), dtype=torch.int8)
    sw = 0.001 * (0.5 + uniform(seed + 1, n))
    x = normal(seed + 2, m, k).to(x_dtype)
    b = normal(seed + 3, n) if bias else None
    w = Int8QTensor.from_int8(qw.cuda(), sw.cuda())
    xd = x.cuda()
    y = int8_gemm(w, quantize_tokens(xd) if packed else xd, bias=None if b is None else b.cuda(), out_dtype=out_dtype)
    sx = scales64(x)
    want, tol = product64(codes64(x, sx), sx, qw, sw, b, out_dtype)
    assert y.dtype == out_dtype
    close(y, want, tol)
    return y


@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 15, 16, 17, 31, 33, 48, 64, 65, 100, 129, 200, 257, 512, 600])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 64), (33, 100), (250, 1024), (1000, 4100), (128, 14336)])
def test_int8_products(m, n, k):
    check_product(m, n, k, seed=m + n)


@pytest.mark.parametrize("x_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("out_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m", [1, 7, 40, 300])
def test_int8_product_types(x_dtype, out_dtype, m):
    check_product(m, 130, 777, x_dtype, out_dtype, bias=m % 2 == 1, packed=m == 7, seed=m)


@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (8, 4096, 14336), (16, 5121, 2050), (203, 5121, 4100), (1030, 2064, 700),
                                   (256, 4096, 4096), (2048, 512, 320), (5000, 48, 64), (3, 128256, 128)])
def test_int8_products_of_many_rows(m, n, k):
    check_product(m, n, k, BF16, F32, bias=True, seed=n)
    check_product(m, n, k, F32, BF16, packed=True, seed=n + 1)


@pytest.mark.parametrize("m", [1, 4, 20, 70, 300])
def test_int8_products_as_whole_numbers(m):
    """Scales of 1: every result is the integer sum, exact in fp32 below 2^24."""
    qw = torch.randint(-9, 10, (300, 1000), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    qx = torch.randint(-9, 10, (m, 1000), generator=torch.Generator().manual_seed(2), dtype=torch.int8)
    w = Int8QTensor.from_int8(qw.cuda(), torch.ones(300, device="cuda"))
    x = Int8QTensor.from_int8(qx.cuda(), torch.ones(m, 1, device="cuda", dtype=BF16))
    assert torch.equal(int8_gemm(w, x).cpu().double(), qx.double() @ qw.double().T)


@pytest.mark.parametrize("m", [1, 17, 130])
def test_int8_products_of_the_largest_codes(m):
    """The longest k of -128 by -128 fills 31 bits."""
    qw = torch.full((18, K_MAX), -128, dtype=torch.int8)
    qx = torch.full((m, K_MAX), -128, dtype=torch.int8)
    qx[-1] = 127
    w = Int8QTensor.from_int8(qw.cuda(), torch.ones(18, device="cuda"))
    x = Int8QTensor.from_int8(qx.cuda(), torch.ones(m, device="cuda"))
    want = torch.full((m, 18), 128.0 * 128 * K_MAX, dtype=torch.float64)
    want[-1] = -128.0 * 127 * K_MAX
    assert torch.equal(int8_gemm(w, x).cpu(), want.float())


@pytest.mark.parametrize("m", [3, 30, 140])
def test_int8_tokens_without_bounds_stay_in_their_token(m):
    w = Int8QTensor.quantize(normal(1, 70, 300).cuda())
    x = normal(2, m, 300)
    clean = int8_gemm(w, x.cuda())
    x[1, 5], x[2, 299] = math.nan, -INF
    y = int8_gemm(w, x.cuda())
    assert torch.isnan(y[1:3]).all()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3:], clean[3:])


def test_int8_product_strides_out_and_shapes():
    w = Int8QTensor.quantize(normal(1, 100, 260).cuda())
    wide = normal(2, 40, 700).cuda()
    for x in (wide[:, 3:263], wide[::2, 101:361], wide[3:4, :260].expand(5, 260), wide.T[:260, :9].T, wide[:0, :260]):
        assert torch.equal(int8_gemm(w, x), int8_gemm(w, x.contiguous()))
        if x.shape[0]:
            assert torch.equal(int8_gemm(w, x), int8_gemm(w, quantize_tokens(x)))
    assert int8_gemm(w, wide[0, :260]).shape == (100,)
    assert torch.equal(int8_gemm(w, wide[0, :260]), int8_gemm(w, wide[:1, :260])[0])
    for m in (1, 9, 30):
        x, room = wide[:m, :260], torch.full((m * 100 + 64,), 7.0, device="cuda", dtype=F16)
        out = room[32:32 + m * 100].view(m, 100)
        assert int8_gemm(w, x, out=out) is out
        assert torch.equal(out, int8_gemm(w, x, out_dtype=F16))
        assert (room[:32] == 7).all() and (room[32 + m * 100:] == 7).all()  # the rows behind the last as they were


def test_int8_same_token_in_any_batch():
    """Sums are integers: a token's results do not depend on the others, nor on how many there are."""
    w = Int8QTensor.quantize(normal(1, 600, 1500).cuda())
    x = normal(2, 700, 1500).cuda()
    whole = int8_gemm(w, x)
    for m in (1, 2, 9, 16, 17, 40, 64, 90, 150, 256, 300, 513):
        assert torch.equal(int8_gemm(w, x[:m]), whole[:m])


def test_int8_refusals():
    w = Int8QTensor.quantize(torch.ones(32, 128, device="cuda"))
    x = torch.ones(4, 128, device="cuda")
    for bad in (dict(x=x[:, :127]), dict(x=x.double()), dict(x=x.cpu()), dict(x=x[None]), dict(x=quantize_tokens(x[:, :64])),
                dict(x=x, bias=torch.ones(31, device="cuda")), dict(x=x, bias=torch.ones(32)),
                dict(x=x, bias=torch.ones(32, device="cuda", dtype=F16)), dict(x=x, out_dtype=torch.int32),
                dict(x=x, out=torch.ones(4, 31, device="cuda")), dict(x=x, out=torch.ones(32, 4, device="cuda").T),
                dict(x=x, out=torch.ones(4, 32, device="cuda"), out_dtype=F16), dict(x=x, out=torch.ones(4, 32)),
                dict(x=x, out=x.view(-1)[:128].view(4, 32)),
                dict(x=x, out=w.data[:512].view(F32).view(4, 32))):
        with pytest.raises(ValueError):
            int8_gemm(w, **bad)
    for codes, scales in ((torch.ones(4, 8, device="cuda"), torch.ones(4, device="cuda")),
                          (torch.ones(4, 8, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda")),
                          (torch.ones(4, 8, dtype=torch.int8, device="cuda"), torch.ones(4)),
                          (torch.ones(0, 8, dtype=torch.int8, device="cuda"), torch.ones(0, device="cuda")),
                          (torch.ones(1, K_MAX + 1, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))):
        with pytest.raises(ValueError):
            Int8QTensor.from_int8(codes, scales)
    with pytest.raises(ValueError):
        Int8QTensor(torch.zeros(100, dtype=torch.uint8, device="cuda"), 16, 64)
    with pytest.raises(ValueError):
        quantize_tokens(torch.ones(1, K_MAX + 1, device="cuda"))


@pytest.mark.parametrize("m", [2, 5, 30])
def test_int8_out_of_another_shape_is_refused(m):
    w = Int8QTensor.quantize(normal(1, 24, 128).cuda())
    x = normal(2, m, 128).cuda()
    for out in (torch.full((24, m), 7.0, device="cuda"), torch.full((m * 24,), 7.0, device="cuda"),
                torch.full((m, 4, 6), 7.0, device="cuda"), torch.full((1, m, 24), 7.0, device="cuda")):
        with pytest.raises(ValueError, match="out must be"):
            int8_gemm(w, x, out=out)
        assert (out == 7).all()
    with pytest.raises(ValueError, match="out must be"):
        int8_gemm(w, x[0], out=torch.empty(1, 24, device="cuda"))
    out = torch.empty(24, device="cuda")
    assert torch.equal(int8_gemm(w, x[0], out=out), int8_gemm(w, x)[0])


@pytest.mark.parametrize("dtype", [F32, F16])
def test_int8_one_token_of_the_longest_k(dtype):
    """Its codes fill most of a workgroup's shared memory."""
    x = normal(3, 1, K_MAX).to(dtype)
    qw = torch.randint(-128, 128, (40, K_MAX), generator=torch.Generator().manual_seed(4), dtype=torch.int8)
    sw = 0.001 * (0.5 + uniform(5, 40))
    y = int8_gemm(Int8QTensor.from_int8(qw.cuda(), sw.cuda()), x.cuda())
    sx = scales64(x)
    close(y, *product64(codes64(x, sx), sx, qw, sw, None, F32))


def test_int8_weights_past_4_gb():
    n, k = 33000, K_MAX  # 4.3 GB of codes
    g = torch.Generator(device="cuda").manual_seed(1)
    qw = torch.cat([torch.randint(-128, 128, (3000, k), generator=g, dtype=torch.int8, device="cuda") for _ in range(11)])
    w = Int8QTensor.from_int8(qw, torch.ones(n, device="cuda"))
    some = torch.tensor([0, 16383, 16384, 32767, 32768, 32999])
    for m in (1, 20, 200):
        x = torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int8, device="cuda")
        y = int8_gemm(w, Int8QTensor.from_int8(x, torch.ones(m, device="cuda")))
        want = x.cpu().double() @ qw[some.cuda()].cpu().double().T
        assert torch.equal(y[:, some.cuda()].cpu(), want.float())


def test_rows_far_apart():
    """Rows whose offsets pass 32 bits."""
    room = torch.empty((1 << 32) + 40000, dtype=F16, device="cuda")
    step = (1 << 31) + 24
    z = normal(1, 2, 3000).to(F16)
    far = room.as_strided((2, 3000), (step, 1), 8)
    far.copy_(z)
    ids, w = route_experts(far[:, :200], 5)
    assert torch.equal(ids.cpu(), route64(z[:, :200], 5)[0])
    weights = Int8QTensor.quantize(normal(2, 50, 3000).cuda())
    assert torch.equal(int8_gemm(weights, far), int8_gemm(weights, z.cuda()))
    u, drafted = uniform(3, 2, 2), torch.randint(0, 3000, (2, 1), generator=torch.Generator().manual_seed(4))
    target, draft = normal(5, 2, 2, 3000).to(F16), normal(6, 2, 1, 3000).to(F16)
    t = room.as_strided((2, 2, 3000), (step, 9000, 1), 4096)
    d = room.as_strided((2, 1, 3000), (step, 1, 1), 24576)
    t.copy_(target)
    d.copy_(draft)
    for dz, given in ((None, None), (draft, d)):
        got, want = verify_draft(t, drafted.cuda(), u.cuda(), given), verify64(target, drafted, u, dz)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_int8_backend_matmul():
    w = Int8QTensor.quantize(normal(1, 48, 96).cuda())
    a = normal(2, 5, 96)
    got = HipBackend().matmul(a.numpy(), w)
    assert np.array_equal(got, int8_gemm(w, a.cuda()).cpu().numpy())


# ---- verify_draft -----------------------------------------------------------------------------

def softmax64(z, temperature):
    z = z.double().numpy() / temperature
    if np.isnan(z).any() or (z == INF).any():
        return None
    if z.max() == -INF:
        return np.zeros_like(z)
    e = np.exp(z - z.max())
    return e / e.sum()


def verify64(target, drafted, u, draft=None, lengths=None, temperature=1.0, draft_temperature=None):
    """One sequence and one draft at a time."""
    seqs, k1, vocab = target.shape
    tokens, accepted = np.full((seqs, k1), -1, dtype=np.int32), np.zeros(seqs, dtype=np.int32)
    for s in range(seqs):
        count = k1 - 1 if lengths is None else min(max(int(lengths[s]), 0), k1 - 1)
        j, weights = 0, None
        while True:
            p = softmax64(target[s, j], temperature)
            d = int(drafted[s, j]) if j < count else -1
            if p is None or not 0 <= d < vocab:
                weights = p
                break
            if draft is None:
                q = np.zeros(vocab)
                q[d] = 1.0
            else:
                q = softmax64(draft[s, j], draft_temperature or temperature)
            if q is None:
                break
            if float(u[s, j]) * q[d] < p[d]:
                tokens[s, j] = d
                j += 1
                continue
            weights = np.maximum(p - q, 0)
            weights = weights if weights.sum() > 0 else p
            break
        accepted[s] = j
        if weights is not None and weights.sum() > 0:
            c = np.cumsum(weights)
            past = np.nonzero((c > float(u[s, -1]) * c[-1]) & (weights > 0))[0]
            tokens[s, j] = past[0] if past.size else np.nonzero(weights)[0][-1]
    return torch.from_numpy(tokens), torch.from_numpy(accepted)


def make_drafts(seqs, k, vocab, dtype=F32, seed=0, draft=True, agree=0.5):
    common = 2.5 * normal(seed, seqs, k + 1, vocab)
    target = (common + agree * normal(seed + 1, seqs, k + 1, vocab)).to(dtype)
    dz = (common[:, :k] + agree * normal(seed + 2, seqs, k, vocab)).to(dtype)
    noise = -torch.log(-torch.log(uniform(seed + 3, seqs, k, vocab).clamp(1e-9, 1 - 1e-7)))
    drafted = (dz.float() + noise).argmax(2) if k else torch.zeros(seqs, 0, dtype=torch.int64)
    return target, drafted, uniform(seed + 4, seqs, k + 1), dz if draft else None


def check_verify(target, drafted, u, draft=None, lengths=None, **kw):
    on = lambda t: None if t is None else t.cuda()  # noqa: E731
    tokens, accepted = verify_draft(target.cuda(), drafted.cuda(), u.cuda(), on(draft), on(lengths), **kw)
    want_tokens, want_accepted = verify64(target, drafted, u, draft, lengths, **kw)
    assert tokens.dtype == accepted.dtype == torch.int32
    assert torch.equal(accepted.cpu(), want_accepted)
    assert torch.equal(tokens.cpu(), want_tokens)
    return want_tokens, want_accepted


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 63, 64, 65, 255, 2047, 2048, 2049, 5000, 32003])
@pytest.mark.parametrize("seqs,k", [(1, 1), (3, 4), (2, 0), (9, 2)])
@pytest.mark.parametrize("draft", [True, False])
def test_verify_draft_sizes(vocab, seqs, k, draft):
    check_verify(*make_drafts(seqs, k, vocab, seed=vocab + seqs, draft=draft))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("draft", [True, False])
def test_verify_draft_types_and_outcomes(dtype, draft):
    seen = set()
    for seed in range(12):
        _, accepted = check_verify(*make_drafts(16, 5, 999, dtype, 10 * seed, draft, agree=0.7), temperature=0.8)
        seen |= set(accepted.tolist())
    # refused everywhere, and nowhere (drafts without probabilities are accepted as often as the target has them)
    assert seen == set(range(6)) if draft else 0 in seen


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_verify_draft_likely_lookups(dtype):
    seen = set()
    for seed in range(12):
        target, drafted, u, _ = make_drafts(16, 5, 999, dtype, 10 * seed)
        drafted = target[:, :5].float().argmax(2)
        _, accepted = check_verify(target, drafted, u, temperature=0.2)
        seen |= set(accepted.tolist())
    assert seen == set(range(6))


@pytest.mark.parametrize("seqs,k,vocab,draft", [(1, 8, 128256, True), (1, 4, 150001, False), (64, 2, 20000, True),
                                                (300, 1, 3000, False), (2, 63, 1000, True), (700, 3, 257, True)])
def test_verify_draft_slices(seqs, k, vocab, draft):
    check_verify(*make_drafts(seqs, k, vocab, BF16 if vocab > 50000 else F32, 3, draft))


def test_verify_draft_lengths_and_ids_that_end_them():
    target, drafted, u, draft = make_drafts(40, 6, 500, seed=5, agree=0.1)
    lengths = torch.randint(-1, 9, (40,), dtype=torch.int32, generator=torch.Generator().manual_seed(1))
    check_verify(target, drafted, u, draft, lengths)
    check_verify(target, drafted, u, None, lengths)
    drafted[::3, 2], drafted[1::3, 0], drafted[2, 5], drafted[5, 1] = -1, 500, 1 << 40, -(1 << 40)
    check_verify(target, drafted, u, draft)
    check_verify(target, drafted.clamp(-5, 600).to(torch.int32), u, draft, lengths)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("vocab", [50, 4111])
def test_verify_draft_masks(draft, vocab):
    target, drafted, u, dz = make_drafts(24, 3, vocab, seed=7, draft=draft)
    allowed = uniform(8, 24, 4, vocab) < 0.1
    allowed[:12].scatter_(2, torch.cat([drafted, drafted[:, :1]], 1)[:12, :, None], True)
    target[~allowed] = -INF
    if draft:
        dz[~(uniform(9, 24, 3, vocab) < 0.5)] = -INF
        dz[20, 1] = -INF
    target[1, 0], target[2, 3], target[3, 1] = -INF, -INF, -INF  # nothing is left
    target[4, 0], target[5, 0] = torch.finfo(F32).min, -INF
    target[5, 0, vocab - 1] = 0.0
    check_verify(target, drafted, u, dz)


@pytest.mark.parametrize("draft", [True, False])
def test_verify_draft_nan_and_infinities_end_a_sequence(draft):
    target, drafted, u, dz = make_drafts(12, 3, 700, seed=11, draft=draft, agree=0.05)
    target[1, 0, 5], target[2, 3, 699], target[3, 1, 0] = math.nan, INF, math.nan
    if draft:
        dz[4, 0, 9], dz[5, 2, 0] = INF, math.nan
    tokens, accepted = check_verify(target, drafted, u, dz)
    assert tokens[1, 0] == -1 and accepted[1] == 0


@pytest.mark.parametrize("vocab", [64, 3001])
def test_verify_draft_equal_distributions(vocab):
    """p = q: every draft with a probability is accepted; one without (its residual is 0 everywhere) falls back to p."""
    target, drafted, u, dz = make_drafts(20, 4, vocab, seed=13)
    dz = target[:, :4].clone()
    _, accepted = check_verify(target, drafted, u, dz)
    assert (accepted == 4).all()
    for s in range(0, 20, 2):
        target[s, 1, drafted[s, 1]] = dz[s, 1, drafted[s, 1]] = -INF
    _, accepted = check_verify(target, drafted, u, dz)
    assert (accepted[::2] == 1).all()


def test_verify_draft_random_numbers_at_the_ends():
    target, drafted, u, dz = make_drafts(8, 2, 900, seed=17)
    last = 1 - 2.0 ** -24
    target[:, :, 0] = -INF  # the first id that may be drawn is not the first
    for a in (0.0, last):
        for b in (0.0, last):
            u[:, :2], u[:, 2] = a, b
            check_verify(target, drafted, u, dz)
            check_verify(target, drafted, u, None)


def test_verify_draft_flat_distributions_by_every_random_number():
    """1024 equal weights: the token is u times 1024, cut, whatever slice it falls into."""
    n = 2048
    u = torch.stack([torch.zeros(n), torch.arange(n) / n], 1)
    target = torch.zeros(1, 2, 1024).expand(n, 2, 1024)
    drafted = torch.zeros(n, 1, dtype=torch.int32)
    tokens, accepted = verify_draft(torch.zeros(1, 2, 1024, device="cuda").expand(target.shape), drafted.cuda(), u.cuda())
    assert (accepted == 1).all()
    assert torch.equal(tokens[:, 1].cpu(), torch.arange(n, dtype=torch.int32) // 2)


@pytest.mark.parametrize("sure", [8.0, 16.0, 30.0])
def test_verify_draft_refuses_a_nearly_certain_lookup(sure):
    """What is left without the draft is a small part of p: its digits come from its own sum."""
    target = normal(19, 6, 2, 3000)
    drafted = torch.randint(0, 3000, (6, 1), generator=torch.Generator().manual_seed(2))
    target[:, :1].scatter_(2, drafted[:, None], 8.0 + sure)
    u = torch.cat([torch.full((6, 1), 1 - 2.0 ** -24), uniform(3, 6, 1)], 1)
    check_verify(target, drafted, u)


@pytest.mark.parametrize("temperature,other", [(1e-3, None), (0.3, 0.9), (4.0, 0.5), (1e3, 1.0), (1e-30, None), (1e30, None)])
def test_verify_draft_temperatures(temperature, other):
    target, drafted, u, dz = make_drafts(10, 3, 1500, seed=23)
    check_verify(target, drafted, u, dz, temperature=temperature, draft_temperature=other)
    check_verify(target, drafted, u, None, temperature=temperature)


def test_verify_draft_large_logits():
    target, drafted, u, dz = make_drafts(6, 2, 600, seed=29)
    check_verify(target * 1e30, drafted, u, dz * 1e30)
    check_verify(target + 1e4, drafted, u, dz - 1e4)


def test_verify_draft_strides():
    target, drafted, u, dz = make_drafts(6, 3, 800, seed=31)
    want = verify64(target, drafted, u, dz)
    wide_t, wide_d = torch.zeros(6, 5, 1001, device="cuda"), torch.zeros(7, 6, 803, device="cuda")
    wide_t[:, 1:, 3:803], wide_d[:3, :6, 1:801] = target.cuda(), dz.transpose(0, 1).cuda()
    wide_i, wide_u = torch.zeros(6, 9, dtype=torch.int64, device="cuda"), torch.zeros(6, 8, device="cuda")
    wide_i[:, 2:5], wide_u[:, 1:5] = drafted.cuda(), u.cuda()
    got = verify_draft(wide_t[:, 1:, 3:803], wide_i[:, 2:5], wide_u[:, 1:5], wide_d[:3, :6, 1:801].transpose(0, 1))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    got = verify_draft(target.transpose(1, 2).contiguous().cuda().transpose(1, 2), drafted.T.contiguous().cuda().T, u.cuda(), dz.cuda())
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    tokens, accepted = verify_draft(torch.empty(0, 3, 5, device="cuda"), torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                                    torch.empty(0, 3, device="cuda"))
    assert tokens.shape == (0, 3) and accepted.shape == (0,)


def test_verify_draft_refusals():
    t, d, u = torch.zeros(2, 4, 9, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, device="cuda")
    good = dict(target=t, drafted=d, uniforms=u)
    for bad in (dict(target=t[0]), dict(target=t.double()), dict(target=t[:, :, :0]), dict(drafted=d[:, :2]), dict(drafted=d.float()),
                dict(drafted=d.cpu()), dict(uniforms=u[:, :3]), dict(uniforms=u.half()), dict(draft=t), dict(draft=t[:, :3].half()),
                dict(draft=t[:, :3].cpu()), dict(lengths=torch.zeros(2, device="cuda")),
                dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(temperature=0.0), dict(temperature=-1.0),
                dict(temperature=math.nan), dict(draft=t[:, :3], draft_temperature=0.0)):
        with pytest.raises(ValueError):
            verify_draft(**{**good, **bad})
    with pytest.raises(ValueError):
        verify_draft(torch.zeros(1, 65, 4, device="cuda"), torch.zeros(1, 64, dtype=torch.int32, device="cuda"), torch.zeros(1, 65, device="cuda"))


# Rows of several pieces a slice (a workgroup takes 2048 logits at a time, 576 rows of 20011 make slices of 6672, 320
# rows of 3336): what the sums are relative to begins with a slice's first logits.

def leading(seqs, k, vocab, lead, temperature, seed):
    """Three ids a row, behind the first 2048, `lead` powers of two over all others."""
    step = temperature * math.log(2)
    target = normal(seed, seqs, k + 1, vocab, scale=0.5 * temperature)
    ids = 2048 + torch.stack([torch.randperm(1200, generator=torch.Generator().manual_seed(seed + 7 + i))[:3]
                              for i in range(seqs * (k + 1))]).view(seqs, k + 1, 3)
    dz = target[:, :k].clone()
    top = lead * step + 0.7 * temperature * normal(seed + 1, seqs, k + 1, 3)
    target.scatter_(2, ids, top)
    dz.scatter_(2, ids[:, :k], top[:, :k] + 0.4 * temperature * normal(seed + 2, seqs, k, 3))
    which = torch.randint(0, 3, (seqs, k, 1), generator=torch.Generator().manual_seed(seed + 3))
    return target, ids[:, :k].gather(2, which)[..., 0], uniform(seed + 4, seqs, k + 1), dz


@pytest.mark.parametrize("temperature", [1.0, 0.05, 0.02, 0.01])
@pytest.mark.parametrize("lead", [40, 61, 130, 300, 520, 700, 890, 910, 2000])
def test_verify_draft_leads_behind_the_first_logits(lead, temperature):
    target, drafted, u, dz = leading(64, 4, 20011, lead, temperature, lead)
    _, accepted = check_verify(target, drafted, u, dz, temperature=temperature)
    assert set(accepted.tolist()) >= {0, 4}
    check_verify(target, drafted, u, None, temperature=temperature)


@pytest.mark.parametrize("temperature", [0.05, 0.03, 0.025, 0.02, 0.015, 0.01])
@pytest.mark.parametrize("vocab", [20011, 32003])
def test_verify_draft_nearly_greedy_batches(temperature, vocab):
    """Likely ids anywhere in rows of ordinary spread."""
    target, _, u, dz = make_drafts(64, 4, vocab, seed=37, agree=0.01)
    ids = torch.randint(0, vocab, (64, 5, 2), generator=torch.Generator().manual_seed(38))
    top = 20.0 + temperature * normal(39, 64, 5, 2)
    target.scatter_(2, ids, top)
    dz.scatter_(2, ids[:, :4], top[:, :4] + 0.3 * temperature * normal(40, 64, 4, 2))
    check_verify(target, ids[:, :4, 0], u, dz, temperature=temperature)
    check_verify(target, ids[:, :4, 0], u, None, temperature=temperature)


@pytest.mark.parametrize("rise", [7, 59, 61, 100, 450, 899, 901, 3000])
def test_verify_draft_rows_that_rise(rise):
    """A whole row a slice (2100 rows), each piece of 2048 `rise` powers of two over the one before, or under it."""
    target, drafted, u, dz = make_drafts(300, 3, 9001, seed=41, agree=0.3)
    for sign in (1, -1):
        up = (sign * rise * math.log(2) * (torch.arange(9001) // 2048)).float()
        at = torch.arange(9001) >= 8192 if sign > 0 else torch.arange(9001) < 2048
        d = torch.where(at, dz, -INF).argmax(2)
        check_verify(target + up, d, u, dz + up)


@pytest.mark.parametrize("temperature,scale", [(1e-30, 1.0), (1e-12, 1.0), (1e-6, 1.0), (1.0, 1e13), (1.0, 1e37), (1e30, 1.0), (1e4, 1e3)])
def test_verify_draft_extremes_of_long_slices(temperature, scale):
    target, drafted, u, dz = make_drafts(64, 4, 20011, seed=43, agree=0.2)
    drafted[::2] = target[::2, :4].argmax(2)
    check_verify(target * scale, drafted, u, dz * scale, temperature=temperature)
    check_verify(target * scale, drafted, u, None, temperature=temperature)


@pytest.mark.parametrize("logit,temperature", [(12.0, 1e-9), (8.0, 1e-9), (-9.0, 1.1e-9), (12.0, 1.2e-8), (3.0, 2e-10)])
def test_verify_draft_neighbours_at_a_low_temperature(logit, temperature):
    """One logit the next float over all others, hundreds of powers of two above them."""
    row = torch.full((20011,), logit)
    row[5000] = torch.nextafter(row[0], torch.tensor(INF))
    u = uniform(45, 300, 2)
    drafted = torch.full((300, 1), 5000)
    target = row.cuda().expand(300, 2, 20011)
    for dz in (None, target[:, :1]):
        tokens, accepted = verify_draft(target, drafted.cuda(), u.cuda(), dz, temperature=temperature)
        assert (tokens.cpu() == 5000).all() and (accepted.cpu() == 1).all()


def test_verify_draft_random_numbers_next_to_a_border():
    """Two ids: the first one's share of the sum is 3e-14 to 6e-13 of itself beside the random number."""
    d = (0.25 + np.arange(1 << 22, dtype=np.float32) * np.float32(2.0 ** -22)).astype(np.float32)
    share = 1 / (1 + np.exp(-d.astype(np.longdouble)))
    u = share.astype(np.float32)
    gap = np.abs(share / u.astype(np.longdouble) - 1).astype(np.float64)
    some = (gap < 6e-13) & (gap > 3e-14) & (u < 1)
    assert some.sum() > 30
    d, u, share = d[some], u[some], share[some]
    target = torch.stack([torch.zeros(d.size), torch.from_numpy(-d)], 1)[:, None]
    tokens, _ = verify_draft(target.cuda(), torch.empty(d.size, 0, dtype=torch.int64, device="cuda"),
                             torch.from_numpy(u)[:, None].cuda())
    assert np.array_equal(tokens[:, 0].cpu().numpy(), (share <= u).astype(np.int32))


# ---- together, on streams and in graphs ---------------------------------------------------

def step_weights():
    w = {"up": Int8QTensor.quantize(normal(1, 512, 256, scale=0.06).cuda()),
         "down": Int8QTensor.quantize(normal(2, 256, 512, scale=0.06).cuda()),
         "router": Int8QTensor.quantize(normal(3, 8, 256, scale=0.1).cuda()),
         "experts": make_experts(8, 256, 256),
         "bias": 0.05 * normal(4, 8).cuda(), "norm": 1 + 0.1 * normal(8, 256).cuda(),
         "head": QTensor.quantize(normal(5, 1024, 256, scale=0.2), ggml.GGML_TYPE_Q4_K, device="cuda")}
    return w


def verify_step(w, x, drafted, u):
    """A verify step's products, experts and decision for one sequence of drafts."""
    _, n = block_norm(x, torch.zeros_like(x), pre_w=w["norm"])
    q = quantize_tokens(n)
    x = x + int8_gemm(w["down"], torch.relu(int8_gemm(w["up"], q)))
    ids, weights = route_experts(int8_gemm(w["router"], q), 2, scores="sigmoid", bias=w["bias"], groups=4, groups_kept=2)
    x = x + moe_grouped_ffn(*w["experts"], x, routing=(ids, weights))[0]
    logits = gemm(w["head"], x)
    tokens, accepted = verify_draft(logits[None], drafted[None], u[None])
    logprobs = token_logprobs(logits, torch.where(tokens[0] >= 0, tokens[0], -1))[0]
    return ids, weights, logits, tokens, accepted, logprobs


def test_a_verify_step_through_all_operators():
    w, x, u = step_weights(), normal(6, 5, 256).cuda(), uniform(7, 5).cuda()
    drafted = torch.randint(0, 1024, (4,), generator=torch.Generator().manual_seed(1)).cuda()
    ids, weights, logits, tokens, accepted, logprobs = verify_step(w, x, drafted, u)
    drafted[:3] = logits[:3].argmax(1)  # likely drafts, and one that is not
    ids, weights, logits, tokens, accepted, logprobs = verify_step(w, x, drafted, u)
    want = verify64(logits.cpu()[None], drafted.cpu()[None], u.cpu()[None])
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(accepted.cpu(), want[1])
    n = int(accepted[0]) + 1
    lp = torch.log_softmax(logits.double(), 1).gather(1, tokens[0, :n, None].long())[:, 0]
    assert (logprobs[:n].double() - lp).abs().max() < 1e-4


def test_captured_verify_steps_replay():
    """Two graphs, replayed in turn on new inputs with eager work between, against eager calls."""
    w = step_weights()
    sets, graphs = [], []
    for i in range(2):
        s = [normal(50 + i, 5, 256).cuda(), torch.randint(0, 1024, (4,)).cuda(), uniform(60 + i, 5).cuda()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            verify_step(w, *s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = verify_step(w, *s)
        sets.append(s)
        graphs.append((g, out))
    for turn in range(4):
        for i, (s, (g, out)) in enumerate(zip(sets, graphs)):
            s[0].copy_(normal(70 + 2 * turn + i, 5, 256))
            s[2].copy_(uniform(80 + 2 * turn + i, 5))
            g.replay()
            want = verify_step(w, *s)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    for g, _ in graphs:  # both in flight, no wait between
        g.replay()
    torch.cuda.synchronize()
    for s, (_, out) in zip(sets, graphs):
        for a, b in zip(out, verify_step(w, *s)):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_captured_calls_of_every_route_replay():
    """Tiles whole and in chunks, the stream of few tokens, residuals, many experts: replayed on new inputs with eager
    work between, against eager calls."""
    w = Int8QTensor.quantize(normal(1, 700, 3000).cuda())
    small = Int8QTensor.quantize(normal(2, 96, 300).cuda())
    experts = make_experts(70, 256, 256)

    def calls(s):
        out = [int8_gemm(w, s["x"][:m]) for m in (1, 9, 40, 300)] + [int8_gemm(small, s["x"][:130, :300], out_dtype=BF16)]
        routing = route_experts(s["z"], 9, scores="sigmoid", bias=s["bias"], groups=7, groups_kept=4, group_score="top2")
        out += [*routing, moe_grouped_ffn(*experts, s["t"], routing=routing)[0]]
        out += verify_draft(s["target"], s["drafted"], s["u"], draft=s["draft"], lengths=s["lengths"])
        return out

    def fill(s, seed):
        for i, name in enumerate(("x", "z", "bias", "t", "target", "draft")):
            s[name].copy_(normal(seed + i, *s[name].shape))
        s["u"].copy_(uniform(seed + 9, *s["u"].shape))
        s["drafted"].copy_(s["draft"].argmax(2))

    s = {"x": torch.empty(300, 3000, device="cuda"), "z": torch.empty(12, 70, device="cuda"), "bias": torch.empty(70, device="cuda"),
         "t": torch.empty(12, 256, device="cuda"), "target": torch.empty(5, 4, 9001, device="cuda"),
         "draft": torch.empty(5, 3, 9001, device="cuda"), "u": torch.empty(5, 4, device="cuda"),
         "drafted": torch.empty(5, 3, dtype=torch.int64, device="cuda"),
         "lengths": torch.tensor([3, 0, 2, 3, 1], dtype=torch.int32, device="cuda")}
    fill(s, 100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = calls(s)
    for turn in range(4):
        fill(s, 200 + 20 * turn)
        g.replay()
        want = calls(s)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once():
    w = step_weights()
    jobs = [[normal(90 + i, 5, 256).cuda(), torch.randint(0, 1024, (4,)).cuda(), uniform(95 + i, 5).cuda()] for i in range(2)]
    want = [verify_step(w, *s) for s in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(verify_step(w, *s))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)
