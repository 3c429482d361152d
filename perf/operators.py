"""Operators around the quantized products of a serving step, measured beside their plain forms.

* ``norm``     -- the seam between two blocks of a decoder: the block's output normalised, gated, scaled and
                  added to the residual stream, and the stream normalised for the next block
                  (``tensor.block_norm``)
* ``logprob``  -- log probabilities of given tokens from the output head's logits, with the entropy and the top
                  alternatives of every row (``tensor.token_logprobs``)
* ``group4``   -- products of a few tokens with 4-bit weights that have one scale (and zero point) per group of
                  32, 64 or 128 along a row (``group4.GroupQTensor``, ``group4.group_gemv``)

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges.  Where ``own`` is false ``run``
computes the plain form with elementary torch operations in float32; where it is true it calls the package.
A decode loop replays a captured graph over its layers, so the cases with ``graph`` do (the package's calls only:
the plain form runs eagerly).  ``exact`` is the definition in float64.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # One token through the 16 seams of eight layers in a decode step's graph, the stream running through.
        {"name": "norm_decode", "op": "norm", "rows": 1, "dim": 4096, "x": "f32", "branch": "f32", "normed": "f32",
         "gate": "none", "scale": 1.0, "layers": 16, "graph": True},
        # A verify batch of 16 tokens in bf16, one learned gate per channel, one call.
        {"name": "norm_verify_bf16", "op": "norm", "rows": 16, "dim": 8192, "x": "bf16", "branch": "bf16",
         "normed": "bf16", "gate": "channel", "scale": 1.0, "layers": 1, "graph": False},
        # A prefill chunk: the products leave fp32, the next GEMM takes fp16; a depth-scaled residual.
        {"name": "norm_prefill", "op": "norm", "rows": 512, "dim": 4096, "x": "f32", "branch": "f32", "normed": "f16",
         "gate": "none", "scale": 0.22, "layers": 1, "graph": False},
        # A long ragged prompt of rows of odd length, one gate per value.
        {"name": "norm_prompt_ragged", "op": "norm", "rows": 7001, "dim": 5121, "x": "f16", "branch": "f32",
         "normed": "f16", "gate": "full", "scale": 1.0, "layers": 1, "graph": False},
        # One sampled token's log probability with the 20 alternatives that an API returns.
        {"name": "logprob_decode", "op": "logprob", "rows": 1, "vocab": 128256, "x": "f32", "tokens": 1, "top": 20,
         "temperature": 1.0, "allowed": 1.0},
        # A constrained step of eight sequences: a grammar leaves one id in a hundred; four candidates each.
        {"name": "logprob_masked", "op": "logprob", "rows": 8, "vocab": 32003, "x": "f16", "tokens": 4, "top": 5,
         "temperature": 0.7, "allowed": 0.01},
        # Scoring a prompt chunk from fp32 logits, the five best alternatives of every position.
        {"name": "logprob_prompt", "op": "logprob", "rows": 512, "vocab": 128256, "x": "f32", "tokens": 1, "top": 5,
         "temperature": 1.0, "allowed": 1.0},
        # A long evaluation in bf16, rows of odd length: only the given tokens and the entropy.
        {"name": "logprob_eval_bf16", "op": "logprob", "rows": 1500, "vocab": 151669, "x": "bf16", "tokens": 1,
         "top": 0, "temperature": 1.0, "allowed": 1.0},
        # One key projection, symmetric, called by itself: the smallest call.
        {"name": "group4_kv", "op": "group4", "m": 1, "n": 1024, "k": 4096, "group": 128, "zeros": False, "x": "f32",
         "layers": 1, "graph": False},
        # The gate and up projections of four layers in a decode step's graph.
        {"name": "group4_decode", "op": "group4", "m": 1, "n": 14336, "k": 4096, "group": 128, "zeros": True,
         "x": "f32", "layers": 8, "graph": True},
        # Speculative verify of eight tokens through the down projections of four layers.
        {"name": "group4_verify", "op": "group4", "m": 8, "n": 4096, "k": 14336, "group": 64, "zeros": True,
         "x": "f16", "layers": 4, "graph": True},
        # Five positions through an output head with small groups.
        {"name": "group4_head", "op": "group4", "m": 5, "n": 128256, "k": 4096, "group": 32, "zeros": False,
         "x": "bf16", "layers": 1, "graph": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "logprob", "group4"])
    if op == "norm":
        rows, dim = _log_int(rng, 1, 8192), _log_int(rng, 512, 8192)
        rows = min(rows, (32 << 20) // dim)
        if rng.random() < 0.6:
            dim = max(512, dim // 256 * 256)
        layers = rng.randint(2, 16) if rows <= 8 else 1
        return {"op": op, "rows": rows, "dim": dim, "x": rng.choice(["f32", "f32", "f16", "bf16"]),
                "branch": rng.choice(["f32", "f32", "f16", "bf16"]), "normed": rng.choice(["f32", "f16", "bf16"]),
                "gate": rng.choice(["none", "none", "channel", "row", "full"]), "scale": rng.choice([1.0, 0.22, 0.5]),
                "layers": layers, "graph": layers > 1}
    if op == "logprob":
        rows, vocab, x = _log_int(rng, 1, 1024), _log_int(rng, 2000, 200000), rng.choice(["f32", "f16", "bf16"])
        rows = max(1, min(rows, (400 << 20) // (vocab * SIZE[x])))
        return {"op": op, "rows": rows, "vocab": vocab, "x": x, "tokens": rng.choice([1, 1, 2, 5]),
                "top": rng.choice([0, 1, 5, 20]), "temperature": rng.choice([1.0, 1.0, 0.6, 1.5]),
                "allowed": rng.choice([1.0, 1.0, 0.5, 0.01])}
    m, n, k = _log_int(rng, 1, 16), _log_int(rng, 256, 65536), _log_int(rng, 512, 16384)
    n = min(n, (256 << 20) // k)
    if rng.random() < 0.7:
        k = max(512, k // 128 * 128)
    layers = rng.randint(2, 8) if n * k <= 32 << 20 else 1
    return {"op": op, "m": m, "n": n, "k": k, "group": rng.choice([32, 64, 128, 128]), "zeros": rng.random() < 0.6,
            "x": rng.choice(["f32", "f16", "bf16"]), "layers": layers, "graph": layers > 1}


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g)


def _uniform(g, *shape):
    return torch.rand(shape, dtype=torch.float32, device="cuda", generator=g)


def _norm_inputs(g, case):
    """A stream with a few large channels, as residual streams have, and the branches of its blocks."""
    rows, dim = case["rows"], case["dim"]
    large = torch.where(_uniform(g, dim) < 0.004, 30.0, 1.0)
    made = {"x": (_normal(g, rows, dim) * large).to(DTYPES[case["x"]]), "seams": []}
    for _ in range(case["layers"]):
        gate = {"none": None, "channel": (dim,), "row": (rows, 1), "full": (rows, dim)}[case["gate"]]
        made["seams"].append({"branch": (0.5 * _normal(g, rows, dim)).to(DTYPES[case["branch"]]),
                              "post": 1 + 0.1 * _normal(g, dim), "pre": 1 + 0.1 * _normal(g, dim),
                              "gate": None if gate is None else torch.sigmoid(_normal(g, *gate)).to(DTYPES[case["branch"]])})
    return made


def _logprob_inputs(g, case):
    """Logits of spread 2.5 with one id per row lifted; given tokens are mostly likely ones, some are padding."""
    rows, vocab, t = case["rows"], case["vocab"], case["tokens"]
    z = _normal(g, rows, vocab).mul_(2.5)
    likely = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)
    z.scatter_add_(1, likely, 18 * _uniform(g, rows, 1))
    other = torch.randint(0, vocab, (rows, t), device="cuda", generator=g)
    u = _uniform(g, rows, t)
    tokens = torch.where(u < 0.6, likely.expand(rows, t), other)
    tokens = torch.where(u > 0.95, -1, tokens)
    z = z.to(DTYPES[case["x"]])
    if case["allowed"] < 1:
        for r in range(0, rows, 64):
            z[r:r + 64].masked_fill_(_uniform(g, min(64, rows - r), vocab) >= case["allowed"], -math.inf)
    return {"logits": z, "tokens": tokens}


def _codes(g, n, k):
    """4-bit codes spread normally around 8, two in a byte, the even one in the low half; an odd row ends in a spare."""
    lut = (8 + 2.7 * torch.erfinv((torch.arange(16, dtype=torch.float64) + 0.5) / 8 - 1) * math.sqrt(2)).round()
    lut = lut.clamp(0, 15).to(torch.uint8).cuda()
    both = (lut[None, :] | (lut[:, None] << 4)).reshape(-1)
    cols, out = (k + 1) // 2, []
    for r in range(0, n, 1 << 15):
        byte = torch.randint(0, 256, (min(1 << 15, n - r), cols), dtype=torch.uint8, device="cuda", generator=g)
        out.append(both[byte.to(torch.int32)])
    return torch.cat(out)


def _group4_inputs(g, case):
    """Weights of spread 0.02 and activations with one value in a thousand twenty times as large."""
    m, n, k = case["m"], case["n"], case["k"]
    groups = -(-k // case["group"])
    x = _normal(g, m, k)
    x = torch.where(_uniform(g, m, k) < 0.001, 20 * x, x).to(DTYPES[case["x"]])
    mats = []
    for _ in range(case["layers"]):
        scales = (0.0074 * (0.8 + 0.4 * _uniform(g, n, groups))).to(torch.float16)
        zeros = torch.randint(6, 10, (n, groups), dtype=torch.uint8, device="cuda", generator=g) if case["zeros"] else None
        mats.append({"packed": _codes(g, n, k), "scales": scales, "zeros": zeros})
    return {"x": x, "mats": mats}


def _inputs(case, seed):
    return {"norm": _norm_inputs, "logprob": _logprob_inputs, "group4": _group4_inputs}[case["op"]](_generator(seed), case)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["graph"] = case, None
    if own and case["op"] == "group4":
        # the layout in HBM that a program keeps its weights in
        from vibeblade_amd.group4 import GroupQTensor
        s["weights"] = [GroupQTensor.from_packed(w["packed"], w["scales"], w["zeros"], k=case["k"], group=case["group"])
                        for w in s.pop("mats")]
    if own and case.get("graph"):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _calls(s)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = _calls(s)
    return s


# ---- the package's calls ---------------------------------------------------------

def _calls(s):
    case = s["case"]
    if case["op"] == "norm":
        from vibeblade_amd.tensor import block_norm
        x, out = s["x"], []
        for seam in s["seams"]:
            x, n = block_norm(x, seam["branch"], post_w=seam["post"], gate=seam["gate"], scale=case["scale"],
                              pre_w=seam["pre"], eps=EPS, normed_dtype=DTYPES[case["normed"]])
            out.append(n)
        return x, out
    if case["op"] == "logprob":
        from vibeblade_amd.tensor import token_logprobs
        return token_logprobs(s["logits"], s["tokens"], top=case["top"], temperature=case["temperature"])
    from vibeblade_amd.group4 import group_gemv
    return [group_gemv(w, s["x"]) for w in s["weights"]]


# ---- the plain forms ---------------------------------------------------------

def _rms(v, w):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w


def _plain_seam(case, x, seam):
    p = _rms(seam["branch"].float(), seam["post"])
    if seam["gate"] is not None:
        p = p * seam["gate"].float()
    y = x.float() + case["scale"] * p
    return y.to(x.dtype), _rms(y, seam["pre"]).to(DTYPES[case["normed"]])


def _plain_norm(s):
    x, out = s["x"], []
    for seam in s["seams"]:
        x, n = _plain_seam(s["case"], x, seam)
        out.append(n)
    return x, out


def _ordered(v):
    """One int64 per value that sorts by value, equal values by the lower index first."""
    bits = (v + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    return (key << 32) - torch.arange(v.shape[1], device=v.device)


def _plain_logprob(s):
    case, tokens = s["case"], s["tokens"]
    v = s["logits"].float()
    top = v.max(1, keepdim=True).values
    d = (v - torch.where(torch.isinf(top), 0.0, top)) * (1 / case["temperature"])
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    entropy = torch.where(total > 0, log_total - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total, 0.0)
    given = (tokens >= 0) & (tokens < case["vocab"])
    lp = torch.where(given, d.gather(1, tokens.clamp(0, case["vocab"] - 1)) - torch.clamp(log_total, min=-3e38), 0.0)
    ids = torch.topk(_ordered(v) if case["top"] else v, case["top"], 1).indices
    best = d.gather(1, ids) - torch.clamp(log_total, min=-3e38)
    return lp, entropy[:, 0], torch.where(torch.isinf(best), -1, ids).to(torch.int32), best


def _plain_product(case, x, w):
    n, k, group = case["n"], case["k"], case["group"]
    q = torch.stack([w["packed"] & 15, w["packed"] >> 4], 2).view(n, -1)[:, :k].float()
    at = torch.arange(k, device=x.device) // group
    zero = 8.0 if w["zeros"] is None else w["zeros"].float()[:, at]
    return x.float() @ ((q - zero) * w["scales"].float()[:, at]).T


def run(state):
    if own:
        if state["graph"] is not None:
            state["graph"].replay()
            return state["out"]
        return _calls(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "logprob":
        return _plain_logprob(state)
    return [_plain_product(state["case"], state["x"], w) for w in state["mats"]]


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    if case["op"] == "norm":
        rows, dim = case["rows"], case["dim"]
        gate = {"none": 0, "channel": dim, "row": rows, "full": rows * dim}[case["gate"]] * SIZE[case["branch"]]
        each = rows * dim * (SIZE[case["branch"]] + SIZE[case["normed"]]) + 8 * dim + gate
        return {"bytes": case["layers"] * each + 2 * rows * dim * SIZE[case["x"]],
                "flops": case["layers"] * 11 * rows * dim}
    if case["op"] == "logprob":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (vocab * SIZE[case["x"]] + 12 * case["tokens"] + 4 + 8 * case["top"]),
                "flops": 6 * rows * vocab}
    m, n, k = case["m"], case["n"], case["k"]
    groups = -(-k // case["group"])
    weights = n * (k / 2 + groups * (2.5 if case["zeros"] else 2))
    return {"bytes": case["layers"] * (weights + 4 * m * n) + m * k * SIZE[case["x"]],
            "flops": case["layers"] * 2 * m * n * k}


# ---- the definitions in float64 ----------------------------------------------------

def _exact_norm(case, s):
    def rms(v, w):
        return w.double() * v / ((v ** 2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()

    x, out = s["x"], []
    for seam in s["seams"]:
        p = rms(seam["branch"].double(), seam["post"])
        y = x.double() + case["scale"] * (p if seam["gate"] is None else seam["gate"].double() * p)
        out.append(rms(y, seam["pre"]))
        x = y.to(s["x"].dtype)  # the stream is stored in its type between the blocks
    return y, out


def _exact_logprob(case, s):
    lps, entropies, tops = [], [], []
    step = max(1, (64 << 20) // case["vocab"])
    for r in range(0, case["rows"], step):
        z = s["logits"][r:r + step].double() / case["temperature"]
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        lp = torch.where(torch.isnan(lp), -math.inf, lp)  # a row that the mask leaves empty
        p = lp.exp()
        entropies.append(torch.where(p > 0, -p * lp, 0.0).sum(1))
        t = s["tokens"][r:r + step]
        known = (t >= 0) & (t < case["vocab"])
        lps.append(torch.where(known, lp.gather(1, torch.where(known, t, 0)), 0.0))
        tops.append(lp.sort(1, descending=True).values[:, :case["top"]].clone())
    return torch.cat(lps), torch.cat(entropies), None, torch.cat(tops)


def _exact_group4(case, s):
    x, out = s["x"].double(), []
    for w in s["mats"]:
        y, step = [], max(1, (1 << 26) // case["k"])
        for r in range(0, case["n"], step):
            byte = w["packed"][r:r + step].to(torch.int16)
            q = torch.empty(byte.shape[0], 2 * byte.shape[1], dtype=torch.float64, device=x.device)
            q[:, 0::2], q[:, 1::2] = byte % 16, byte // 16
            q = q[:, :case["k"]]
            z = w["zeros"][r:r + step].double() if w["zeros"] is not None else torch.full_like(w["scales"][r:r + step], 8, dtype=torch.float64)
            spread = lambda v: v.double().repeat_interleave(case["group"], 1)[:, :case["k"]]  # noqa: E731
            y.append(x @ (spread(w["scales"][r:r + step]) * (q - spread(z))).T)
        out.append(torch.cat(y, 1))
    return out


def exact(case, seed):
    return {"norm": _exact_norm, "logprob": _exact_logprob, "group4": _exact_group4}[case["op"]](case, _inputs(case, seed))
