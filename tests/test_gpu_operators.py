"""block_norm, token_logprobs and the 4-bit group products on the GPU against
their definitions in float64.

Tolerances count roundings.  U = 2^-24 is half a step of fp32; a stored value
may be half a step of its own type off (finfo.eps / 2 relative, or half the
smallest subnormal).  A sum of n values in T chains and a tree adds at most
n / T + 16 roundings relative to the sum of their magnitudes.
"""
import math

import numpy as np
import pytest
import torch

from vibeblade_amd import _lib, ggml
from vibeblade_amd.group4 import GroupQTensor, group_gemv
from vibeblade_amd.quant import pack_nibbles
from vibeblade_amd.tensor import QTensor, activation, block_norm, embed_rows, gemm, token_logprobs

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


def half_step(want, dtype):
    """Half a step of `dtype` at `want`."""
    f = torch.finfo(dtype)
    return want.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def close(got, want, tol):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    assert not torch.isnan(got[~torch.isnan(want)]).any()
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin].nan_to_num(7e77), want[~fin].nan_to_num(7e77))
    off = (got - want).abs()[fin] - tol.expand(want.shape)[fin]
    assert off.numel() == 0 or off.max() <= 0, f"{off.max():.3e} over the tolerance"


# ---- block_norm ------------------------------------------------------------------

def norm64(x, b, post, gate, scale, pre, eps):
    """(y, n) and the magnitude that y's roundings are relative to."""
    x, p = x.double(), b.double()
    if post is not None:
        p = p / ((p * p).mean(-1, keepdim=True) + eps).sqrt() * post.double()
    if gate is not None:
        p = p * gate.double()
    p = scale * p
    y = x + p
    r = 1 / ((y * y).mean(-1, keepdim=True) + eps).sqrt()
    return y, None if pre is None else y * r * pre.double(), x.abs() + p.abs(), r


def check_norm(x, b, post, gate, scale, pre, eps, y, n):
    cpu = lambda t: None if t is None else t.cpu()  # noqa: E731
    x, b, post, gate, pre = map(cpu, (x, b, post, gate, pre))
    wy, wn, mag, r = norm64(x, b, post, gate, scale, pre, eps)
    # half of the sum's roundings and 16 single ones go into p and y; mean(y^2) has a sum of its own and y's
    c = x.shape[-1] / 256 / 2 + 16
    close(y, wy, c * U * mag + half_step(wy, y.dtype))
    if pre is None:
        assert n is None
        return
    rough = c * U * (mag.square().mean(-1, keepdim=True).sqrt() * r)  # of the norm, relative
    w = pre.double().abs()
    close(n, wn, (c * U * mag * r * w + (rough + c * U) * wn.abs()) + half_step(wn, n.dtype))


DIMS = [1, 2, 3, 7, 64, 255, 1000, 1024, 2049, 4096, 5121, 8192, 14336, 16384, 40000]


@pytest.mark.parametrize("dim", DIMS)
def test_block_norm_lengths(dim):
    rows = 3
    x, b = normal(dim, rows, dim, scale=3).cuda(), normal(dim + 1, rows, dim).cuda()
    post, pre = (1 + normal(dim + 2, dim, scale=0.1)).cuda(), (1 + normal(dim + 3, dim, scale=0.1)).cuda()
    y, n = block_norm(x, b, post_w=post, pre_w=pre, scale=0.5)
    check_norm(x, b, post, None, 0.5, pre, 1e-5, y, n)


@pytest.mark.parametrize("dim", [5, 256, 257, 1025, 2048, 2050, 4095, 4097, 6145, 8191, 8193, 10241, 12287, 14337])
@pytest.mark.parametrize("gate", [None, "full"])
def test_block_norm_many_rows(dim, gate):
    """More rows than CUs, lengths at and beside the borders of the pieces of a row."""
    rows = 300
    x, b = normal(dim, rows, dim, scale=3).cuda(), normal(dim + 1, rows, dim, dtype=F16).cuda()
    post, pre = (1 + normal(dim + 2, dim, scale=0.1)).cuda(), (1 + normal(dim + 3, dim, scale=0.1)).cuda()
    g = normal(dim + 4, rows, dim, dtype=BF16).cuda() if gate else None
    y, n = block_norm(x, b, post_w=post, gate=g, pre_w=pre, normed_dtype=BF16)
    check_norm(x, b, post, g, 1.0, pre, 1e-5, y, n)


@pytest.mark.parametrize("rows,dims", [
    (1100, [4, 5, 257, 512, 513, 768, 769, 1024, 1025, 1536, 1537, 2048, 2049, 2560, 2561, 3000, 3100, 4096, 4097, 5120, 5121,
            5632, 5633, 6144, 6145, 6657, 7168, 7169]),
    (400, [300, 1024, 1100, 2000, 2049, 4096, 4100, 6144, 14336]),
    (2, [257, 1025, 4097, 8192, 8193, 12288, 12289, 14337, 16383, 16385])])
def test_block_norm_rows_by_waves(rows, dims):
    """Each number of waves and pieces that a row may take, in place and with a gate of each row."""
    for dim in dims:
        x, b = normal(dim, rows, dim, scale=2, dtype=BF16).cuda(), normal(dim + 1, rows, dim).cuda()
        post, pre = (1 + normal(dim + 2, dim, scale=0.1)).cuda(), (1 + normal(dim + 3, dim, scale=0.1)).cuda()
        g = normal(dim + 4, rows, 1, dtype=F16).cuda()
        was = x.clone()
        y, n = block_norm(x, b, post_w=post, gate=g, pre_w=pre, normed_dtype=F16, out=x)
        assert y.data_ptr() == x.data_ptr()
        check_norm(was, b, post, g, 1.0, pre, 1e-5, y, n)


def test_block_norm_stores_special_values_in_16_bits():
    """What a narrow type holds of NaN, infinities, overflow and ties: as torch rounds."""
    v = torch.tensor([[math.nan, INF, -INF, 3.4e38, -3.4e38, 1.0 + 2 ** -8, 1.0 + 3 * 2 ** -8, 1.0 + 2 ** -11, 65519.0,
                       65520.0, 1e-40, -1e-40, 2.0 ** -25, 0.0, -0.0, 7.0]])
    for dtype in (F16, BF16):
        # (a stream of 16 bits in, the branch brings the value in fp32)
        y, _ = block_norm(torch.zeros(1, 16, dtype=dtype, device="cuda"), v.cuda())
        want = (v + 0.0).to(dtype)
        assert torch.equal(y.cpu().isnan(), want.isnan())
        assert torch.equal(y.cpu().nan_to_num(5), want.nan_to_num(5))


@pytest.mark.parametrize("xt", [F32, F16, BF16])
@pytest.mark.parametrize("bt", [F32, F16, BF16])
@pytest.mark.parametrize("nt", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [512, 771])
def test_block_norm_types(xt, bt, nt, dim):
    x, b = normal(1, 5, dim, scale=2, dtype=xt).cuda(), normal(2, 5, dim, dtype=bt).cuda()
    post, pre = (1 + normal(3, dim, scale=0.1)).cuda(), (1 + normal(4, dim, scale=0.1)).cuda()
    gate = torch.sigmoid(normal(5, 5, dim)).to(bt).cuda()
    y, n = block_norm(x, b, post_w=post, gate=gate, pre_w=pre, eps=1e-6, normed_dtype=nt)
    assert y.dtype == xt and n.dtype == nt
    check_norm(x, b, post, gate, 1.0, pre, 1e-6, y, n)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "row", "full", "one", "strided"])
@pytest.mark.parametrize("rows,dim", [(1, 4096), (4, 1001)])
def test_block_norm_parts(post, pre, gate, rows, dim):
    x, b = normal(1, rows, dim).cuda(), normal(2, rows, dim).cuda()
    pw, qw = (1 + normal(3, dim)).cuda() if post else None, (1 + normal(4, dim)).cuda() if pre else None
    g = None if gate is None else {
        "channel": normal(5, dim), "row": normal(5, rows, 1), "full": normal(5, rows, dim), "one": normal(5, 1),
        "strided": normal(5, rows, 2 * dim)[:, ::2]}[gate].cuda()
    y, n = block_norm(x, b, post_w=pw, gate=g, scale=-0.7, pre_w=qw)
    check_norm(x, b, pw, None if g is None else g.expand(rows, dim), -0.7, qw, 1e-5, y, n)


def test_block_norm_strides_offsets_and_leading_axes():
    wide = normal(1, 6, 700).cuda()
    x, b = wide[:, 1:514], normal(2, 6, 3, 513).cuda()[:, 1]
    post, pre = normal(3, 513).cuda(), normal(4, 513).cuda()
    out = torch.full((6, 601), 7.0, device="cuda")
    y, n = block_norm(x, b, post_w=post, pre_w=pre, out=out[:, 3:516])
    assert y.data_ptr() == out[:, 3:].data_ptr()
    check_norm(x, b, post, None, 1.0, pre, 1e-5, y, n)
    assert bool((out[:, :3] == 7).all()) and bool((out[:, 516:] == 7).all())
    x3, b3 = normal(5, 2, 3, 96).cuda(), normal(6, 2, 3, 96, dtype=F16).cuda()
    y3, n3 = block_norm(x3, b3, pre_w=post[:96], gate=normal(7, 2, 1, 1).cuda())
    assert y3.shape == n3.shape == (2, 3, 96)
    check_norm(x3, b3, None, normal(7, 2, 1, 1).expand(2, 3, 96), 1.0, post[:96], 1e-5, y3, n3)
    # one row repeated for all (stride 0), a transposed branch
    row = normal(8, 1, 128).cuda().expand(5, 128)
    bt = normal(9, 128, 5).cuda().t()
    y, n = block_norm(row, bt, pre_w=post[:128])
    check_norm(row, bt, None, None, 1.0, post[:128], 1e-5, y, n)


@pytest.mark.parametrize("dim", [4096, 4097, 50000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_block_norm_in_place(dim, dtype):
    x, b = normal(1, 9, dim, dtype=dtype).cuda(), normal(2, 9, dim, dtype=dtype).cuda()
    post, pre = normal(3, dim).cuda(), normal(4, dim).cuda()
    y0, n0 = block_norm(x, b, post_w=post, pre_w=pre)
    y1, n1 = block_norm(x, b, post_w=post, pre_w=pre, out=x)
    assert y1 is x and torch.equal(y0, x) and torch.equal(n0, n1)


def test_block_norm_empty_zero_and_unbounded_rows():
    y, n = block_norm(torch.empty(0, 64, device="cuda"), torch.empty(0, 64, device="cuda"), pre_w=torch.ones(64))
    assert y.shape == n.shape == (0, 64)
    x, b, one = torch.zeros(4, 300, device="cuda"), torch.zeros(4, 300, device="cuda"), torch.ones(300, device="cuda")
    x[1, 5], b[2, 7], x[3, 299] = float("nan"), INF, -INF
    y, n = block_norm(x, b, post_w=one, pre_w=one)
    assert not y[0].any() and not n[0].any()  # a row of zeros stays one
    assert torch.isnan(n[1]).all() and torch.isnan(y[2, 7]) and y[3, 299] == -INF
    assert torch.isfinite(y[0]).all() and torch.isnan(n[3, 299])
    y, n = block_norm(x[:1], b[:1], post_w=one, pre_w=one, eps=0.0)
    assert torch.isnan(y).all()  # 0 / 0, as the formula says


def test_block_norm_refusals():
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for kw in (dict(branch=x[:, :32]), dict(branch=x[:3]), dict(branch=x.double()), dict(branch=x.cpu()),
               dict(post_w=w[:32]), dict(pre_w=torch.ones(65)), dict(gate=w[:32]), dict(gate=w.double()),
               dict(gate=w.cpu()), dict(gate=torch.ones(2, 4, 64, device="cuda")), dict(out=x[:3]), dict(out=x.half()),
               dict(out=torch.zeros(64, 4, device="cuda").t()), dict(out=x[:1].expand(4, 64)), dict(eps=-1.0),
               dict(pre_w=w, normed_dtype=torch.float64)):
        with pytest.raises(ValueError):
            block_norm(x, **{"branch": x, **kw})
    for bad in (x.double(), x.int(), torch.zeros((), device="cuda"), torch.zeros(3, 0, device="cuda")):
        with pytest.raises(ValueError):
            block_norm(bad, bad)


# ---- token_logprobs ----------------------------------------------------------------

def logprobs64(z, tokens, top, temperature):
    """The definition in float64: (lp, entropy, ids, best) and the rows' tolerances."""
    z = z.cpu()
    v = z.double() / temperature
    rows, vocab = v.shape
    m = v.max(1, keepdim=True).values
    bad = (torch.isnan(v) | (v == INF)).any(1, keepdim=True)
    empty = (v == -INF).all(1, keepdim=True)
    d = v - torch.where(torch.isinf(m), 0.0, m)
    e = torch.where(bad, 0.0, d.exp())
    s = e.sum(1, keepdim=True) - torch.where(empty | bad, 0.0, 1.0)  # exact enough: checked apart where it is small
    t = torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True)
    rest = torch.log1p(s)
    lp = torch.where(empty, -INF, d - rest)
    h = torch.where(empty, 0.0, rest - t / (1 + s))
    lp, h = torch.where(bad, math.nan, lp), torch.where(bad, math.nan, h)
    # exp's argument has 3 roundings, exp 4; a lane's chain is at most vocab / 64 + 16 long
    spread = -t / (1 + s)
    tol_s = (3 * spread + 4 + vocab / 64 + 16) * U
    tol_lp = tol_s + 4 * U * d.abs().nan_to_num(0, 0, 0)
    tol_h = 2 * tol_s + (3 * torch.where(e > 0, e * d * d, 0.0).sum(1, keepdim=True) / (1 + s)
                         + (vocab / 64 + 24) * spread) * U
    key = torch.where(torch.isnan(z.double()), -INF, z.double())
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top]
    ids = torch.where(key.gather(1, order) == -INF, -1, order)
    best = torch.where(ids < 0, -INF, lp.gather(1, order))
    best = torch.where(bad, math.nan, best)
    out = None
    if tokens is not None:
        tk = tokens.cpu().reshape(rows, -1)
        inside = (tk >= 0) & (tk < vocab)
        at = torch.where(inside, tk, 0).long()
        out = torch.where(inside, lp.gather(1, at), 0.0), tol_lp.gather(1, at)
    return out, (h, tol_h), ids, (best, tol_lp.gather(1, order))


def check_logprobs(z, tokens, top=0, temperature=1.0):
    lp, h, ids, best = token_logprobs(z, tokens, top=top, temperature=temperature)
    z2 = z.reshape(1, -1) if z.dim() == 1 else z
    want, (wh, th), wids, (wbest, tbest) = logprobs64(z2, tokens, top, temperature)
    if want is not None:
        assert lp.shape == tokens.shape
        close(lp.reshape(want[0].shape), *want)
    close(h, wh[:, 0], th[:, 0])
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long(), wids)
    close(best, wbest, tbest)


def pick(seed, rows, t, vocab):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (rows, t), generator=g).cuda()


VOCABS = [1, 2, 3, 63, 64, 65, 257, 1000, 4095, 8193, 32003, 128256]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("rows", [1, 3])
def test_token_logprobs_lengths(vocab, rows):
    z = normal(vocab, rows, vocab, scale=3).cuda()
    check_logprobs(z, pick(1, rows, 2, vocab), top=min(5, vocab))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 50001), (2, 4097), (40, 3001), (300, 777), (1030, 130)])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_token_logprobs_types_rows_and_tops(dtype, rows, vocab, top):
    z = normal(7, rows, vocab, scale=2.5, dtype=dtype).cuda()  # 16-bit types: many equal logits
    check_logprobs(z, pick(2, rows, 1, vocab), top=top, temperature=0.7)


@pytest.mark.parametrize("rows,vocab", [(600, 20011), (1100, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_token_logprobs_many_long_rows(rows, vocab, dtype):
    z = normal(3, rows, vocab, scale=2, dtype=dtype).cuda()
    check_logprobs(z, pick(3, rows, 1, vocab), top=7)


@pytest.mark.parametrize("order", ["up", "down", "equal", "two"])
@pytest.mark.parametrize("vocab", [100, 5000, 70001])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_token_logprobs_orders_and_ties(order, vocab, top):
    i = torch.arange(vocab, dtype=F32)
    row = {"up": i * 1e-3, "down": -i * 1e-3, "equal": torch.full((vocab,), -2.5),
           "two": torch.where(i % 977 == 5, 1.0, 0.0)}[order]
    z = torch.stack([row, row.flip(0), -row]).cuda()
    check_logprobs(z, pick(4, 3, 1, vocab), top=top)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(4, 333), (4, 40000), (520, 5000)])
def test_token_logprobs_masks(dtype, rows, vocab):
    """Rows with nothing, one id, three ids and the type's lowest value left by the mask."""
    z = normal(5, rows, vocab, scale=2, dtype=dtype)
    z[0] = -INF
    z[1, 1:] = -INF
    z[2, torch.arange(vocab) % 111 != 7] = -INF
    z[2, 333:] = -INF
    z[3, 3:] = torch.finfo(dtype).min
    tokens = torch.zeros(rows, 3, dtype=torch.int32)
    tokens[:, 1], tokens[:, 2] = vocab - 1, 7
    check_logprobs(z.cuda(), tokens.cuda(), top=9, temperature=1.3)


@pytest.mark.parametrize("vocab", [50, 30000])
def test_token_logprobs_nan_and_infinities(vocab):
    z = normal(6, 5, vocab)
    z[1, vocab // 2], z[2, vocab - 1], z[3, :2] = float("nan"), INF, INF
    z[4] = float("nan")
    check_logprobs(z.cuda(), pick(5, 5, 1, vocab), top=4)


def test_token_logprobs_certain_token_keeps_its_digits():
    """log p = -log1p(S) with S near 1e-9: a sum that holds the maximum's 1 would give 0."""
    for vocab in (1000, 60000):
        z = torch.full((2, vocab), -30.0)
        z[:, 17] = torch.tensor([0.0, 3.0])
        lp, h, _, best = token_logprobs(z.cuda(), torch.tensor([17, 17]).cuda(), top=1)
        s = (vocab - 1) * torch.tensor([-30.0, -33.0], dtype=torch.float64).exp()
        want = -torch.log1p(s)
        tol = want.abs() * (3 * 33 + 4 + vocab / 64 + 16) * U
        close(lp, want, tol)
        close(best[:, 0], want, tol)
        d = torch.tensor([30.0, 33.0], dtype=torch.float64)
        close(h, torch.log1p(s) + s * d / (1 + s), (tol * 36) * 2)


def test_token_logprobs_given_tokens_padding_and_strides():
    wide = normal(8, 6, 3001).cuda()
    z = wide[:, 1:2500]
    tokens = torch.tensor([0, 2498, -1, 2499, 1 << 40, 5]).cuda()
    check_logprobs(z, tokens, top=3)
    assert token_logprobs(z, tokens)[0][2:5].tolist() == [0.0, 0.0, 0.0]
    check_logprobs(z, pick(6, 6, 8, 2499)[:, ::2].to(torch.int32), top=1)
    check_logprobs(normal(9, 2001).cuda(), torch.tensor([[4, 2000, -7]]).cuda(), top=2)
    check_logprobs(normal(9, 1, 500).cuda().expand(4, 500), pick(7, 4, 1, 500), top=2)
    check_logprobs(normal(10, 500, 4).cuda().t(), pick(7, 4, 1, 500), top=2)
    check_logprobs(normal(9, 3, 500).cuda(), None, top=2)
    for dt in (F16, BF16):  # rows that start at an odd element
        check_logprobs(normal(11, 5, 4099, dtype=dt).cuda()[:, 1:4098], pick(8, 5, 1, 4097), top=5)
    e = token_logprobs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), top=3)
    assert [tuple(t.shape) for t in e] == [(0,), (0,), (0, 3), (0, 3)]


@pytest.mark.parametrize("temperature", [1e-6, 0.1, 25.0, 1e12])
def test_token_logprobs_temperatures(temperature):
    z = normal(12, 3, 5000, scale=2).cuda()
    check_logprobs(z, pick(9, 3, 2, 5000), top=6, temperature=temperature)


def test_token_logprobs_refusals():
    z, t = torch.zeros(4, 10, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for args, kw in (((z, t[:3]), {}), ((z, t.float()), {}), ((z, t.cpu()), {}), ((z.double(), t), {}),
                     ((z, t), dict(top=11)), ((z, t), dict(top=-1)), ((z, t), dict(temperature=0.0)),
                     ((z, t.view(1, 4)), {}), ((z.view(2, 2, 10), t), {}), ((torch.zeros(4, 0, device="cuda"), t), {}),
                     ((torch.zeros(4, 100, device="cuda"), t), dict(top=65))):
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)


# ---- 4-bit weights with group scales ---------------------------------------------------

def parts(seed, rows, k, group, zeros):
    """Random codes, scales and zero points on the host, and the weights in float64."""
    rng = np.random.default_rng(seed)
    groups = -(-k // group)
    q = rng.integers(0, 16, (rows, k), dtype=np.uint8)
    s = (rng.uniform(0.5, 1.5, (rows, groups)) * 0.01 * rng.choice([-1, 1], (rows, groups))).astype(np.float16)
    z = rng.integers(0, 16, (rows, groups), dtype=np.uint8) if zeros else None
    at = np.arange(k) // group
    w = (q.astype(np.float64) - (8.0 if z is None else z[:, at])) * s.astype(np.float64)[:, at]
    packed = np.stack([pack_nibbles(r) for r in q])
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    return dev(packed), dev(s), dev(z), torch.from_numpy(w)


def check_product(w, w64, x, y):
    """Activations keep 22 bits or more below a block's largest (digits) or are exact (fp16 operands); a group's sum
    is exact, or one chain of instructions of 32 products each."""
    x64 = x.cpu().double().reshape(-1, w64.shape[1])
    mag = x64.abs() @ w64.abs().T
    want = x64 @ w64.T
    close(y.reshape(want.shape), want, (4 * U + (w64.shape[1] / 32 + 32) * U) * mag)


SHAPES = [(1, 1), (1, 128), (15, 7), (16, 128), (17, 129), (33, 96), (64, 1000), (100, 256), (130, 4096), (48, 5001),
          (20, 14336), (16, 20000)]


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("zeros", [False, True])
def test_group4_decode_is_exact(rows, k, group, zeros):
    packed, s, z, w64 = parts(rows + k, rows, k, group, zeros)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=group)
    assert w.shape == (rows, k) and w.zeros == zeros
    assert torch.equal(w.dequantize().cpu().double(), w64)


@pytest.mark.parametrize("rows,k", SHAPES)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False), (384, True)])
@pytest.mark.parametrize("m,dtype", [(1, F32), (1, F16), (1, BF16), (2, F32), (5, BF16), (8, F32), (9, F32), (16, F16),
                                     (17, F16), (33, F32)])
def test_group4_products(rows, k, group, zeros, m, dtype):
    packed, s, z, w64 = parts(rows * 3 + k, rows, k, group, zeros)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=group)
    x = normal(m, m, k, dtype=dtype).cuda()
    y = group_gemv(w, x if m > 1 else x[0])
    assert y.dtype == F32 and y.shape == ((m, rows) if m > 1 else (rows,))
    check_product(w, w64, x, y)


@pytest.mark.parametrize("rows", [1023, 4096, 14336, 32000])
@pytest.mark.parametrize("m", [1, 4, 16, 70])
def test_group4_products_of_many_rows(rows, m):
    k = 512
    packed, s, z, w64 = parts(rows, rows, k, 64, True)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=64)
    x = normal(m, m, k, dtype=F16 if m == 16 else F32).cuda()
    check_product(w, w64, x, group_gemv(w, x))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m", [1, 3, 8])
def test_group4_activations_of_every_size(dtype, m):
    """Outliers, tiny and huge values, a row of zeros, subnormals: each block of 128 keeps its own precision."""
    k = 1024
    packed, s, z, w64 = parts(5, 40, k, 128, True)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=128)
    top, low = (60000.0, 1e-7) if dtype == F16 else (3e37, 1e-37)
    x = normal(6, m, k)
    x[0, 128:256] *= low
    x[0, 256:384] *= top / 8
    x[0, 400] = 3000.0
    x[0, 512:640] = 0
    x[-1, 700:] = 0
    x = x.to(dtype).cuda()
    y = group_gemv(w, x)
    x64 = x.cpu().double()
    # per block of 128: 22 bits of each value or 2^-38 of the block's largest, then as check_product
    b = x64.abs().view(m, -1, 128).max(2, keepdim=True).values.expand(m, -1, 128).reshape(m, k)
    mag = x64.abs() @ w64.abs().T
    close(y, x64 @ w64.T, (4 * U + (k / 32 + 32) * U) * mag + 2.0 ** -38 * (b @ w64.abs().T))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m", [5, 6, 16])
@pytest.mark.parametrize("zeros", [False, True])
def test_group4_subnormal_activations(dtype, m, zeros):
    """Every value below the type's smallest normal one; those are fp32's own subnormals in bf16."""
    packed, s, z, w64 = parts(9, 40, 512, 64, zeros)
    w = GroupQTensor.from_packed(packed, s, z, k=512, group=64)
    f = torch.finfo(dtype)
    x = (torch.from_numpy(np.random.default_rng(m).integers(-100, 101, (m, 512))).double() * (f.tiny * f.eps)).to(dtype)
    assert (x != 0).any() and x.abs().double().max() < f.tiny
    y = group_gemv(w, x.cuda())
    mag = x.double().abs() @ w64.abs().T
    close(y, x.double() @ w64.T, (4 * U + (512 / 32 + 32) * U) * mag + 2.0 ** -146)  # and sixteen roundings below the normal range


def test_group4_activations_of_a_few_tokens_without_bounds_stay_in_theirs():
    packed, s, z, w64 = parts(7, 50, 300, 64, True)
    w = GroupQTensor.from_packed(packed, s, z, k=300, group=64)
    for dtype in (F16, BF16):
        x = normal(8, 9, 300, dtype=dtype)
        x[1, 7], x[2, 299] = float("nan"), INF
        y = group_gemv(w, x.cuda()).cpu()
        assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
        rest = [0, 3, 4, 5, 6, 7, 8]
        check_product(w, w64, x[rest], y[rest])


def test_group4_activations_without_bounds_stay_in_their_token():
    packed, s, z, w64 = parts(7, 50, 300, 64, True)
    w = GroupQTensor.from_packed(packed, s, z, k=300, group=64)
    for dtype in (F32, F16, BF16):
        x = normal(8, 4, 300, dtype=dtype)
        x[1, 7], x[2, 299] = float("nan"), INF
        y = group_gemv(w, x.cuda()).cpu()
        assert torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
        for t in (0, 3):
            check_product(w, w64, x[t:t + 1], y[t:t + 1])


def test_group4_strides_offsets_and_out():
    packed, s, z, w64 = parts(9, 70, 257, 32, True)
    w = GroupQTensor.from_packed(packed, s, z, k=257, group=32)
    for dtype in (F32, F16, BF16):
        wide = normal(10, 5, 400, dtype=dtype).cuda()
        check_product(w, w64, wide[:, 3:260], group_gemv(w, wide[:, 3:260]))
        check_product(w, w64, wide[2, 1:258], group_gemv(w, wide[2, 1:258]))
        check_product(w, w64, wide[:1, :257].expand(3, 257), group_gemv(w, wide[:1, :257].expand(3, 257)))
        t = normal(11, 257, 4, dtype=dtype).cuda().t()
        check_product(w, w64, t, group_gemv(w, t))
    x = normal(12, 2, 257).cuda()
    buf = torch.full((142,), 7.0, device="cuda")
    y = group_gemv(w, x, out=buf[1:141])
    check_product(w, w64, x, y)
    assert buf[0] == 7 and buf[141] == 7
    assert group_gemv(w, torch.empty(0, 257, device="cuda")).shape == (0, 70)
    # parts with strides of their own pack the same
    w2 = GroupQTensor.from_packed(packed.t().contiguous().t(), s.t().contiguous().t(), z.t().contiguous().t(), k=257, group=32)
    assert torch.equal(w.data, w2.data)


def test_group4_same_call_same_bits():
    packed, s, z, _ = parts(13, 500, 4096, 128, True)
    w = GroupQTensor.from_packed(packed, s, z, k=4096, group=128)
    x = normal(14, 3, 4096).cuda()
    y = group_gemv(w, x)
    for _ in range(5):
        assert torch.equal(y, group_gemv(w, x))


@pytest.mark.parametrize("group", [32, 64, 128, 640])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_group4_quantize(group, zeros, dtype):
    """Each weight within half a step of its group (its scale rounded to fp16 first), groups of zeros exact."""
    rows, k = 20, 1283
    src = normal(15, rows, k, scale=0.02, dtype=dtype)
    src[3, :group] = 0
    src[4, 5] = 0.5
    w = GroupQTensor.quantize(src.cuda(), group=group, zeros=zeros)
    v, got = src.double(), w.dequantize().cpu().double()
    assert not got[3, :group].any()
    for g in range(-(-k // group)):
        a, q = v[:, g * group:(g + 1) * group], got[:, g * group:(g + 1) * group]
        lo, hi = a.min(1, keepdim=True).values.clamp(max=0), a.max(1, keepdim=True).values.clamp(min=0)
        step = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7
        # half a step to the nearest code and, with a rounded zero point, half a step past the range's ends; the
        # scale in fp16 moves 15 (7) steps by 2^-11 each
        tol = step * ((1.0 if zeros else 0.5) + 16 * 2.0 ** -11 + 1e-5) + 2.0 ** -24 * 16
        assert bool(((a - q).abs() <= tol).all())


def test_group4_refusals():
    packed, s, z, _ = parts(16, 20, 100, 32, True)
    good = dict(packed=packed, scales=s, zeros=z, k=100, group=32)
    for kw in (dict(k=99 - 1), dict(k=103), dict(k=0), dict(group=48), dict(group=64), dict(scales=s.float()),
               dict(scales=s[:, :3]), dict(zeros=z[:19]), dict(zeros=z.int()), dict(zeros=z.cpu()),
               dict(packed=packed.int()), dict(packed=packed[:0]), dict(packed=packed.cpu()), dict(scales=None)):
        with pytest.raises(ValueError):
            GroupQTensor.from_packed(**{**good, **kw})
    w = GroupQTensor.from_packed(**good)
    x = torch.zeros(2, 100, device="cuda")
    for bad in (x[:, :99], x.double(), x.cpu(), x.view(1, 2, 100), x.int()):
        with pytest.raises(ValueError):
            group_gemv(w, bad)
    for out in (torch.zeros(39, device="cuda"), torch.zeros(40, device="cuda").half(), torch.zeros(40)):
        with pytest.raises(ValueError):
            group_gemv(w, x, out=out)
    for kw in (dict(rows=33), dict(k=300), dict(group=33), dict(zeros=False)):  # 33: a row tile more than 20
        with pytest.raises(ValueError):
            GroupQTensor(w.data, **{**dict(rows=20, k=100, group=32, zeros=True), **kw})
    with pytest.raises(ValueError):
        GroupQTensor.quantize(torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        GroupQTensor.quantize(torch.zeros(4, 64, device="cuda"), group=40)


def test_group4_backend_matmul():
    from vibeblade_amd.gpu import GPUBackend
    packed, s, z, w64 = parts(17, 24, 160, 32, True)
    w = GroupQTensor.from_packed(packed, s, z, k=160, group=32)
    a = normal(18, 3, 160)
    check_product(w, w64, a, torch.from_numpy(GPUBackend().matmul(a.numpy(), w)))
    with pytest.raises(ValueError):
        GPUBackend().matmul(a.numpy()[:, :100], w)


# ---- together, on streams and in graphs ---------------------------------------------------

class Step:
    """A decode step's FFN half with the three operators and the GGUF ops beside them: embedding rows, the seam
    into the block, gate / up / down with group scales, the seam out, the output head, log probabilities."""
    H, I, V = 256, 512, 1000

    def __init__(self, seed):
        self.table = QTensor.quantize(normal(seed, self.V, self.H), ggml.GGML_TYPE_Q8_0, device="cuda")
        make = lambda n, rows, k: GroupQTensor.quantize(normal(seed + n, rows, k, scale=k ** -0.5).cuda(), group=64)  # noqa: E731
        self.gate, self.up, self.down = make(1, self.I, self.H), make(2, self.I, self.H), make(3, self.H, self.I)
        self.head = make(4, self.V, self.H)
        self.w = [(1 + normal(seed + 5 + i, self.H, scale=0.1)).cuda() for i in range(4)]

    def __call__(self, tokens, branch, targets):
        x = embed_rows(self.table, tokens)
        x, n = block_norm(x, branch, post_w=self.w[0], pre_w=self.w[1], scale=0.5)
        h = activation(group_gemv(self.gate, n), 0) * group_gemv(self.up, n)
        x, n = block_norm(x, group_gemv(self.down, h), post_w=self.w[2], pre_w=self.w[3])
        return (x,) + token_logprobs(group_gemv(self.head, n), targets, top=4)

    def exact(self, tokens, branch, targets):
        x = self.table.dequantize()[tokens.long()].cpu().double()
        w = [v.cpu() for v in self.w]
        x, n, _, _ = norm64(x, branch.cpu(), w[0], None, 0.5, w[1], 1e-5)
        d = lambda q: q.dequantize().cpu().double().T  # noqa: E731
        g = n @ d(self.gate)
        x, n, _, _ = norm64(x, (g * torch.sigmoid(g) * (n @ d(self.up))) @ d(self.down), w[2], None, 1.0, w[3], 1e-5)
        lp = torch.log_softmax(n @ d(self.head), 1)
        return x, lp.gather(1, targets.cpu()[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp.sort(1, descending=True)

    def inputs(self, seed, t):
        return pick(seed, 1, t, self.V)[0].to(torch.int32), normal(seed, t, self.H).cuda(), pick(seed + 1, 1, t, self.V)[0]


def far_rows(t, apart=1_200_000_000):
    """t's rows, 2.4 GB apart (16-bit types): the third begins behind 2^31 elements and 2^32 bytes."""
    buf = torch.empty((t.shape[0] - 1) * apart + t.shape[1], dtype=t.dtype, device="cuda")
    far = buf.as_strided(t.shape, (apart, 1))
    far.copy_(t)
    return far


def test_rows_far_apart():
    x, b = normal(1, 3, 5003, dtype=BF16), normal(2, 3, 5003, dtype=F16)
    pre = (1 + normal(3, 5003, scale=0.1)).cuda()
    fx, fb = far_rows(x), far_rows(b)
    y, n = block_norm(fx, fb, pre_w=pre, out=fx)
    check_norm(x, b, None, None, 1.0, pre, 1e-5, y, n)
    z, tok = normal(4, 3, 9001, scale=4, dtype=F16), torch.tensor([0, 9000, 77])
    check_logprobs(far_rows(z), tok.cuda(), top=3)
    packed, s, zp, w64 = parts(5, 40, 5003, 128, True)
    w = GroupQTensor.from_packed(packed, s, zp, k=5003, group=128)
    for dtype in (F16, BF16):
        v = normal(6, 3, 5003, dtype=dtype)
        check_product(w, w64, v, group_gemv(w, far_rows(v)))


def test_group4_weights_past_4_gb():
    k, rows, last = 16384, 560000, 48
    packed, s, z, w64 = parts(11, last, k, 64, True)
    small = GroupQTensor.from_packed(packed, s, z, k=k, group=64)
    data = torch.zeros(small.nbytes // last * rows, dtype=torch.uint8, device="cuda")
    data[-small.nbytes:] = small.data
    assert data.numel() > 2 ** 32
    w = GroupQTensor(data, rows, k, 64, True)
    for m, dtype in ((1, F32), (2, BF16), (9, F16)):
        x = normal(m, m, k, dtype=dtype).cuda()
        y = group_gemv(w, x)
        assert (y[:, :-last] == 0).all()
        check_product(small, w64, x, y[:, -last:])


def test_logits_of_one_row_for_all():
    z = normal(21, 1, 4099, scale=4)
    tok = torch.arange(700, dtype=torch.int32).reshape(-1, 1).cuda()
    check_logprobs(z.cuda().expand(700, 4099), tok, top=2)


@pytest.mark.parametrize("m,dtype", [(1, F32), (2, BF16), (6, F32), (9, F16), (9, BF16)])
def test_group4_products_over_a_very_long_k(m, dtype):
    """More chunks of k than one launch holds at a time."""
    k = 262144 + 100
    packed, s, z, w64 = parts(m, 20, k, 128, True)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=128)
    x = normal(m, m, k, dtype=dtype).cuda()
    check_product(w, w64, x, group_gemv(w, x))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
def test_group4_chunks_of_k_fit(dtype, group, zeros):
    """Every number of blocks of k near those that a workgroup holds, for each number of tokens."""
    for m in range(1, 17):
        for blocks in (9, 10, 11, 15, 17, 18, 19, 21, 33, 34, 35, 37, 41, 51, 67, 68, 69, 103, 137, 205):
            k = 256 * blocks - blocks % 3
            data = torch.randint(0, 256, (_lib.load().vb_group4_bytes(20, k, group, zeros),), dtype=torch.uint8,
                                 device="cuda", generator=torch.Generator("cuda").manual_seed(blocks)) & 0x3b  # finite scales
            w = GroupQTensor(data, 20, k, group, zeros)
            x = torch.randn(m, k, device="cuda", generator=torch.Generator("cuda").manual_seed(m)).to(dtype)
            w64, x64 = w.dequantize().double(), x.double()
            off = (group_gemv(w, x).double() - x64 @ w64.T).abs() - (k / 32 + 36) * U * (x64.abs() @ w64.abs().T)
            assert off.max() <= 0, (m, blocks)


@pytest.mark.parametrize("dim", [300, 5121, 16385, 40000])
def test_block_norm_of_the_stream_itself(dim):
    x, pre = normal(dim, 5, dim).cuda(), (1 + normal(1, dim, scale=0.1)).cuda()
    was = x.clone()
    y, n = block_norm(x, x, post_w=pre, pre_w=pre, scale=0.5, out=x)
    check_norm(was, was, pre, None, 0.5, pre, 1e-5, y, n)


def test_group4_refuses_out_over_x():
    packed, s, z, _ = parts(3, 128, 128, 32, False)
    w = GroupQTensor.from_packed(packed, s, z, k=128, group=32)
    buf = torch.zeros(400, device="cuda")
    for x, out in ((buf[:128], buf[:128]), (buf[:128], buf[100:228]), (buf[100:228], buf[:128]),
                   (buf[:384].view(3, 128)[:, :], buf[:384].view(3, 128))):
        with pytest.raises(ValueError, match="overlaps"):
            group_gemv(w, x, out=out)
    group_gemv(w, buf[:128], out=buf[128:256])
    group_gemv(w, buf[:0].view(0, 128), out=buf[:0].view(0, 128))


@pytest.mark.parametrize("t", [1, 5])
def test_a_step_through_all_operators(t):
    """fp32 throughout: each product and norm is within 150 roundings of its terms' magnitudes, which are at most
    about eight times the results, over seven operators: 1e4 U."""
    step = Step(100)
    args = step.inputs(200, t)
    x, lp, h, ids, best = step(*args)
    wx, wlp, wh, (wbest, wids) = step.exact(*args)
    for got, want in ((x, wx), (lp, wlp), (h, wh), (best, wbest[:, :4])):
        close(got, want, 1e4 * U * (want.abs() + 1))
    assert torch.equal(ids.cpu().long(), wids[:, :4])


def test_head_of_gguf_weights_feeds_the_log_probabilities():
    """gemm's logits of a Q6_K head, as a scoring loop has them."""
    head = QTensor.quantize(normal(1, 700, 512, scale=0.05), ggml.GGML_TYPE_Q6_K, device="cuda")
    x, b = normal(2, 6, 512).cuda(), normal(3, 6, 512).cuda()
    _, n = block_norm(x, b, pre_w=torch.ones(512, device="cuda"), normed_dtype=F16)
    z = gemm(head, n)
    check_logprobs(z, pick(4, 6, 1, 700), top=5)


@pytest.mark.parametrize("t", [1, 5])
def test_captured_steps_replay(t):
    """Two graphs of the same kind, replayed in turn on new inputs with eager work between, against eager calls."""
    steps = [Step(300), Step(400)]
    sets = [s.inputs(500 + i, t) for i, s in enumerate(steps)]
    graphs = []
    for s, args in zip(steps, sets):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s(*args)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = s(*args)
        graphs.append((g, out))
    for turn in range(4):
        for i, (s, args, (g, out)) in enumerate(zip(steps, sets, graphs)):
            for a, new in zip(args, s.inputs(600 + 10 * turn + i, t)):
                a.copy_(new)
            g.replay()
            for got, want in zip([v.clone() for v in out], s(*args)):
                assert torch.equal(got, want)
    for g, _ in graphs:  # both in flight, no wait between
        g.replay()
    torch.cuda.synchronize()
    for s, args, (_, out) in zip(steps, sets, graphs):
        for got, want in zip(out, s(*args)):
            assert torch.equal(got, want)


def test_calls_on_two_streams_at_once():
    step = Step(700)
    sets = [step.inputs(800 + i, 3) for i in range(4)]
    want = [step(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, a in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append([step(*a) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("temperature", [1e-7, 1e-8, 3e-9, 1e-9, 1e-12, 1e-20, 1e-25, 1e-29, 1e-30])
@pytest.mark.parametrize("rows,vocab,top", [(3, 20000, 6), (40, 4096, 0), (600, 3001, 3)])
def test_token_logprobs_low_temperatures(temperature, rows, vocab, top):
    """Near-greedy sampling: log2(e) / T times a logit passes 2^31, and its rounding any exponent that fp32 holds.
    (A temperature that fp32 holds, so that its own rounding is none of the result's.)"""
    z = normal(31, rows, vocab, scale=3)
    z[1, 7] = z[1, vocab - 2] = z[1].max()  # two places of the maximum
    check_logprobs(z.cuda(), pick(31, rows, 2, vocab), top=top, temperature=float(np.float32(temperature)))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fill", [-1e9, -1e10, -1e15, -1e20, -1e30, 8e9])
@pytest.mark.parametrize("rows,vocab,top", [(5, 333, 4), (5, 40000, 9), (5, 40000, 0), (520, 5000, 9)])
def test_token_logprobs_finite_masks(dtype, fill, rows, vocab, top):
    """Rows that an additive mask leaves at a large finite value: all of them, but for one, but for the last few,
    but for a stretch in between, and every second."""
    for temperature in (1.0, 0.75, 0.3, 0.1):
        z = normal(32, rows, vocab, scale=2, dtype=dtype)
        z[0] = fill
        z[1, torch.arange(vocab) != vocab // 3] = fill
        z[2, :vocab - 20] = fill
        z[3, :vocab // 4] = fill
        z[3, vocab // 2:] = fill
        z[4, ::2] = fill
        tokens = torch.tensor([[0, vocab // 3, vocab - 1, vocab // 2 - 1]]).expand(rows, 4)
        check_logprobs(z.cuda(), tokens.cuda(), top=top, temperature=float(np.float32(temperature)))


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("exponent", [20, 22, 23, 24, 25, 26])
@pytest.mark.parametrize("vocab", [300, 9000, 50001])
def test_token_logprobs_far_from_zero(sign, exponent, vocab):
    """Logits whose common part, times log2(e), is a power of two with many places left behind the point: whichever
    way the sums are kept, terms on both sides of the border count."""
    step = 2.0 ** (exponent - 24)
    base = round(sign * 2.0 ** exponent * math.log(2) / step) * step
    off = (normal(33, 4, vocab, scale=2) / step).round() * step
    off[1], off[2] = off[1].sort().values, off[2].sort(descending=True).values
    off[3] = torch.linspace(-6, 6, vocab).div(step).round() * step
    z = (base + off.double()).float()
    for top in (0, 5):
        check_logprobs(z.cuda(), pick(34, 4, 3, vocab), top=top)


@pytest.mark.parametrize("dim", [300, 771, 5121, 16385, 40000])
@pytest.mark.parametrize("rows", [1, 5, 300, 1100])
def test_block_norm_over_the_branch_or_the_gate(dim, rows):
    if rows * dim > 6 << 20:
        rows = 40
    x, b, g = normal(1, rows, dim).cuda(), normal(2, rows, dim).cuda(), normal(3, rows, dim).cuda()
    post, pre = (1 + normal(4, dim, scale=0.1)).cuda(), (1 + normal(5, dim, scale=0.1)).cuda()
    want = block_norm(x, b, post_w=post, gate=g, pre_w=pre)
    for over in (x, b, g):
        kept = over.clone()
        y, n = block_norm(x, b, post_w=post, gate=g, pre_w=pre, out=over)
        assert y is over and torch.equal(y, want[0]) and torch.equal(n, want[1])
        over.copy_(kept)


def test_block_norm_in_columns_of_one_buffer():
    """x, branch, gate and out side by side in a wider buffer: their ranges of memory meet, their rows do not."""
    wide = normal(6, 7, 4 * 130).cuda()
    x, b, g, out = (wide[:, i * 130:(i + 1) * 130] for i in range(4))
    pre = (1 + normal(7, 130, scale=0.1)).cuda()
    want = block_norm(x, b, post_w=pre, gate=g, pre_w=pre)
    y, n = block_norm(x, b, post_w=pre, gate=g, pre_w=pre, out=out)
    assert torch.equal(y, want[0]) and torch.equal(n, want[1])
    with pytest.raises(ValueError, match="overlaps"):
        block_norm(x, b, out=wide[:, 129:259])


def test_block_norm_gates_of_few_values_at_any_stride():
    for rows, dim in ((1, 1), (4, 1), (0, 64), (1, 64)):
        x, b = normal(1, rows, dim).cuda(), normal(2, rows, dim).cuda()
        pre = (1 + normal(3, dim, scale=0.1)).cuda()
        for gate in (normal(4, rows, 5 * dim).cuda()[:, ::5], normal(5, 5 * dim).cuda()[::5]):
            y, n = block_norm(x, b, gate=gate, pre_w=pre)
            check_norm(x, b, None, gate.expand(rows, dim), 1.0, pre, 1e-5, y, n)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 128])
def test_group4_quantize_keeps_what_is_no_number(dtype, zeros, group):
    """A NaN or an infinity has no code: its group is NaN, and no other one changes."""
    src = normal(41, 9, 300, scale=0.02, dtype=dtype)
    want = GroupQTensor.quantize(src.cuda(), group=group, zeros=zeros).dequantize().cpu()
    bad = {(1, 0): math.nan, (2, group - 1): INF, (3, group): -INF, (4, 299): math.nan, (5, 298): INF}
    for (r, c), v in bad.items():
        src[r, c] = v
        want[r, c // group * group:(c // group + 1) * group] = math.nan
    src[6, 4], src[6, 5] = INF, -INF
    want[6, :group] = math.nan
    w = GroupQTensor.quantize(src.cuda(), group=group, zeros=zeros)
    got = w.dequantize().cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
    for m, xt in ((1, F32), (3, BF16), (8, F16)):
        y = group_gemv(w, normal(m, m, 300, dtype=xt).cuda()).cpu()
        assert y[:, 1:7].isnan().all() and y[:, [0, 7, 8]].isfinite().all()


def test_group4_refuses_zero_points_past_four_bits():
    packed, s, z, _ = parts(16, 20, 100, 32, True)
    z[19, 3] = 16
    with pytest.raises(ValueError, match="zero points"):
        GroupQTensor.from_packed(packed, s, z, k=100, group=32)
    z[19, 3] = 15
    GroupQTensor.from_packed(packed, s, z, k=100, group=32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("m", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_group4_small_activations_beside_large_ones(dtype, m, group, zeros):
    """Each output is one activation times one weight (every other code is the zero point), so what is lost of a
    value beside an outlier of its block of 128 is seen by itself.  With `big` the block's largest magnitude: fp32 is
    exact from 2^-6 big on and below within 2^-30 big, 16-bit digits from 2^-14 (bf16) or 2^-11 (fp16) on and within
    2^-22, fp16 operands throughout, bf16 ones brought to fp16 from 2^-31 on and within 2^-38."""
    k = 384
    rng = np.random.default_rng(m)
    z = rng.integers(0, 16, (k, -(-k // group)), dtype=np.uint8) if zeros else None
    at = np.arange(k) // group
    q = (z[:, at] if zeros else np.full((k, k), 8)).astype(np.int64)
    diag = np.arange(k)
    own = q[diag, diag]
    q[diag, diag] = np.where(own < 8, own + 3, own - 3)
    s = np.full((k, -(-k // group)), 0.5, dtype=np.float16)
    packed = np.stack([pack_nibbles(r.astype(np.uint8)) for r in q])
    w = GroupQTensor.from_packed(torch.from_numpy(packed).cuda(), torch.from_numpy(s).cuda(),
                                 torch.from_numpy(z).cuda() if zeros else None, k=k, group=group)
    gain = torch.from_numpy(np.where(own < 8, 1.5, -1.5))
    small = 2.0 ** -14 if dtype == F16 else 2.0 ** -30
    x = normal(m, m, k) * torch.from_numpy(small ** rng.uniform(0, 1, (m, k))).float()
    x[:, 200] = torch.from_numpy(rng.uniform(500, 4000, m)).float()  # the second block's outlier
    x[:, 256:] *= 2.0 ** -6                                          # the third has its own scale
    x = x.to(dtype)
    as_fp16 = m > 5 or (dtype == F16 and m > 2)
    exact, lost = {F32: (6, 30), F16: (99, 99) if as_fp16 else (11, 22), BF16: (31, 38) if as_fp16 else (14, 22)}[dtype]
    v = x.double()
    big = v.abs().view(m, 3, 128).amax(2, keepdim=True).expand(m, 3, 128).reshape(m, k)
    tol = torch.where(v.abs() >= 2.0 ** -exact * big, 0.0, 2.0 ** -lost * big) + 8 * U * v.abs()
    close(group_gemv(w, x.cuda()), v * gain, tol * 1.5)
    if lost < 99:  # a few bits fewer would be seen
        step = 2.0 ** (4 - lost) * big.log2().floor().exp2()
        assert (((v / step).round() * step - v).abs() > tol).any()


@pytest.mark.parametrize("dtype,m", [(F32, 1), (F32, 2), (F32, 9), (BF16, 3), (BF16, 8)])
@pytest.mark.parametrize("zeros", [False, True])
def test_group4_largest_activations(dtype, m, zeros):
    """Up to the range that the header gives: 4 sum |W| max |x| just below 2^128."""
    k = 384
    packed, s, z, w64 = parts(61, 40, k, 128, zeros)
    w = GroupQTensor.from_packed(packed, s, z, k=k, group=128)
    x = normal(62, m, k).double()
    top = x.abs().view(m, 3, 128).amax(2)  # per block
    bound = 4 * torch.einsum("nb,mb->mn", w64.abs().view(40, 3, 128).sum(2), top).amax(1, keepdim=True)
    x = (x * (0.98 * 2.0 ** 128 / bound)).to(dtype)
    y = group_gemv(w, x.cuda())
    assert y.isfinite().all()
    check_product(w, w64, x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [30, 9000])
def test_token_logprobs_of_opposite_ends_of_the_range(dtype, vocab):
    """z - max leaves fp32's range where the log probability, over a temperature, does not."""
    z = normal(71, 2, vocab, scale=1e38).clamp(-3e38, 3e38).to(dtype)
    z[0, 3], z[0, 20], z[1, 7], z[1, 8] = 3.2e38, -3.2e38, -3.2e38, 3.3e38
    for temperature in (4.0, 1024.0, float(np.float32(1e30))):
        check_logprobs(z.cuda(), torch.tensor([[3, 20, 5], [7, 8, 1]]).cuda(), top=20, temperature=temperature)
