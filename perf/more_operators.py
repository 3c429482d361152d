"""Operators of a speculative step through a model of experts, measured beside their plain forms.

* ``route``   -- experts of every token from the router's logits: softmax or sigmoid scores, a bias that balances
                 the load, groups of experts, top-k, renormalised weights (``tensor.route_experts``)
* ``int8``    -- products in 8-bit integers with a scale per token and one per output channel
                 (``int8.Int8QTensor``, ``int8.quantize_tokens``, ``int8.int8_gemm``)
* ``verify``  -- drafted tokens against the target's probabilities, from given random numbers, and the token that
                 follows them (``tensor.verify_draft``)

``listed()`` names the cases, ``draw(rng)`` gives others of the same ranges.  Where ``own`` is false ``run``
computes the plain form with elementary torch operations; where it is true it calls the package.  A decode loop
replays a captured graph over its layers, so the cases with ``graph`` do (the package's calls only: the plain
form runs eagerly).  ``exact`` is the definition in float64.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # One token's router, called by itself.
        {"name": "route_decode", "op": "route", "tokens": 1, "experts": 128, "topk": 8, "x": "f32",
         "scores": "softmax", "bias": False, "groups": 1, "kept": 1, "group_score": "max", "renorm": True,
         "scale": 1.0, "masked": 0.0, "layers": 1, "graph": False},
        # The routers of twelve layers in the graph of a verify step of 16 tokens; balanced by a bias, groups of 32.
        {"name": "route_verify", "op": "route", "tokens": 16, "experts": 256, "topk": 8, "x": "f32",
         "scores": "sigmoid", "bias": True, "groups": 8, "kept": 4, "group_score": "top2", "renorm": True,
         "scale": 2.5, "masked": 0.0, "layers": 12, "graph": True},
        # A ragged prefill chunk in bf16, where equal logits are common; probabilities as they are.
        {"name": "route_chunk", "op": "route", "tokens": 777, "experts": 160, "topk": 6, "x": "bf16",
         "scores": "softmax", "bias": False, "groups": 8, "kept": 3, "group_score": "max", "renorm": False,
         "scale": 16.0, "masked": 0.0, "layers": 1, "graph": False},
        # The prompts of a whole batch.
        {"name": "route_prefill", "op": "route", "tokens": 16384, "experts": 256, "topk": 8, "x": "f32",
         "scores": "sigmoid", "bias": True, "groups": 8, "kept": 4, "group_score": "top2", "renorm": True,
         "scale": 2.5, "masked": 0.0, "layers": 1, "graph": False},
        # One key projection, called by itself: the smallest call.
        {"name": "int8_kv", "op": "int8", "m": 1, "n": 1024, "k": 4096, "x": "f32", "out": "f32", "bias": False,
         "shared": False, "layers": 1, "graph": False},
        # The gate and up projections of four layers in a decode step's graph.
        {"name": "int8_decode", "op": "int8", "m": 1, "n": 14336, "k": 4096, "x": "bf16", "out": "bf16", "bias": False,
         "shared": False, "layers": 8, "graph": True},
        # Speculative verify of eight tokens through the down projections of four layers.
        {"name": "int8_verify", "op": "int8", "m": 8, "n": 4096, "k": 14336, "x": "f16", "out": "f32", "bias": False,
         "shared": False, "layers": 4, "graph": True},
        # A short ragged chunk through a projection of odd sizes with a bias.
        {"name": "int8_chunk_ragged", "op": "int8", "m": 203, "n": 5121, "k": 4100, "x": "f32", "out": "f32",
         "bias": True, "shared": False, "layers": 1, "graph": False},
        # A long prompt through gate and up, which share the quantized tokens.
        {"name": "int8_prefill", "op": "int8", "m": 4096, "n": 14336, "k": 4096, "x": "bf16", "out": "bf16",
         "bias": False, "shared": True, "layers": 2, "graph": False},
        # One sequence whose drafts were looked up in its own text: no probabilities come with them.
        {"name": "verify_lookup", "op": "verify", "seqs": 1, "drafts": 4, "vocab": 128256, "x": "f32", "draft": False,
         "ragged": False, "temperature": 1.0, "allowed": 1.0},
        # Eight sequences with drafts of different lengths by a draft model, half precision, an odd vocabulary.
        {"name": "verify_ragged", "op": "verify", "seqs": 8, "drafts": 5, "vocab": 32003, "x": "f16", "draft": True,
         "ragged": True, "temperature": 0.7, "allowed": 1.0},
        # A full batch with a draft model.
        {"name": "verify_batch", "op": "verify", "seqs": 64, "drafts": 4, "vocab": 128256, "x": "f32", "draft": True,
         "ragged": False, "temperature": 1.0, "allowed": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "int8", "verify"])
    if op == "route":
        tokens, groups = _log_int(rng, 1, 16384), rng.choice([1, 1, 4, 8])
        experts = max(2, _log_int(rng, 8, 256) // groups) * groups
        kept = rng.randint(max(1, groups // 4), groups)
        topk = min(rng.choice([1, 2, 4, 6, 8]), kept * (experts // groups))
        layers = rng.randint(2, 12) if tokens <= 16 else 1
        return {"op": op, "tokens": tokens, "experts": experts, "topk": topk, "x": rng.choice(["f32", "f16", "bf16"]),
                "scores": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups,
                "kept": kept, "group_score": rng.choice(["max", "top2"]), "renorm": rng.random() < 0.6,
                "scale": rng.choice([1.0, 2.5, 16.0]), "masked": rng.choice([0.0, 0.0, 0.1]), "layers": layers,
                "graph": layers > 1}
    if op == "int8":
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 256, 32768), _log_int(rng, 256, 16384)
        n = min(n, (64 << 20) // k)
        m = max(1, min(m, int(4.8e11) // (n * k)))
        if rng.random() < 0.6:
            k = max(256, k // 128 * 128)
        layers = rng.randint(2, 8) if m <= 16 and n * k <= 32 << 20 else 1
        return {"op": op, "m": m, "n": n, "k": k, "x": rng.choice(["f32", "f16", "bf16"]),
                "out": rng.choice(["f32", "f16", "bf16"]), "bias": rng.random() < 0.3, "shared": rng.random() < 0.3,
                "layers": layers, "graph": layers > 1}
    seqs, drafts, vocab = _log_int(rng, 1, 64), rng.randint(1, 8), _log_int(rng, 2000, 150000)
    x, draft = rng.choice(["f32", "f32", "f16", "bf16"]), rng.random() < 0.6
    seqs = max(1, min(seqs, (295 << 20) // ((drafts + 1) * vocab * SIZE[x] * (2 if draft else 1))))
    return {"op": op, "seqs": seqs, "drafts": drafts, "vocab": vocab, "x": x, "draft": draft,
            "ragged": rng.random() < 0.4, "temperature": rng.choice([1.0, 1.0, 0.6, 1.5]),
            "allowed": rng.choice([1.0, 1.0, 0.5, 0.02])}


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(shape, dtype=torch.float32, device="cuda", generator=g)


def _uniform(g, *shape):
    return torch.rand(shape, dtype=torch.float32, device="cuda", generator=g)


def _route_inputs(g, case):
    """Logits of spread 1.5 over experts of which some are liked by all tokens; the bias lowers those."""
    tokens, experts, made = case["tokens"], case["experts"], []
    for _ in range(case["layers"]):
        liked = _normal(g, experts)
        z = 1.5 * _normal(g, tokens, experts) + liked
        if case["masked"]:
            z = torch.where(_uniform(g, tokens, experts) < case["masked"], -math.inf, z)
        made.append({"logits": z.to(DTYPES[case["x"]]),
                     "bias": -0.1 * liked + 0.02 * _normal(g, experts) if case["bias"] else None})
    return {"routers": made}


def _int8_inputs(g, case):
    """Weights that fill the codes' range as a channel's maximum over 127 leaves them; activations of spread 1 with
    one value in a thousand twenty times as large."""
    m, n, k = case["m"], case["n"], case["k"]
    x = _normal(g, m, k)
    x = torch.where(_uniform(g, m, k) < 0.001, 20 * x, x).to(DTYPES[case["x"]])
    lut = (32 * torch.erfinv((torch.arange(65536, dtype=torch.float64) + 0.5) / 32768 - 1) * math.sqrt(2)).round()
    lut = lut.clamp(-127, 127).to(torch.int8).cuda()
    mats = []
    for _ in range(case["layers"]):
        rows = [lut[torch.randint(0, 65536, (min(4096, n - r), k), dtype=torch.int32, device="cuda", generator=g)]
                for r in range(0, n, 4096)]
        mats.append({"codes": torch.cat(rows), "scales": 0.0006 * (0.8 + 0.4 * _uniform(g, n)),
                     "bias": _normal(g, n) if case["bias"] else None})
    return {"x": x, "mats": mats}


def _verify_inputs(g, case):
    """A draft model's logits and a target that mostly agrees with them; drafts sampled from the former, or, where
    none come with them, mostly likely tokens.  A grammar leaves a share of the ids."""
    b, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    kind = DTYPES[case["x"]]
    target = torch.empty((b, k + 1, vocab), dtype=kind, device="cuda")
    draft = torch.empty((b, k, vocab), dtype=kind, device="cuda") if case["draft"] else None
    drafted = torch.empty((b, k), dtype=torch.int64, device="cuda")
    for s in range(b):
        common = 2.5 * _normal(g, k + 1, vocab)
        likely = torch.randint(0, vocab, (k + 1, 6), device="cuda", generator=g)
        common.scatter_add_(1, likely, 6 + 8 * _uniform(g, k + 1, 6))
        if case["allowed"] < 1:
            allowed = _uniform(g, k + 1, vocab) < case["allowed"]
            common = torch.where(allowed.scatter(1, likely, True), common, -math.inf)
        target[s] = (common + 0.4 * _normal(g, k + 1, vocab)).to(kind)
        if draft is not None:
            draft[s] = (common[:k] + 0.4 * _normal(g, k, vocab)).to(kind)
            noise = -torch.log(-torch.log(_uniform(g, k, vocab).clamp(1e-12, 1 - 1e-7)))
            drafted[s] = (draft[s].float() / case["temperature"] + noise).argmax(1)
        else:
            other = torch.randint(0, vocab, (k,), device="cuda", generator=g)
            drafted[s] = torch.where(_uniform(g, k) < 0.8, target[s, :k].float().argmax(1), other)
    lengths = torch.randint(0, k + 1, (b,), dtype=torch.int32, device="cuda", generator=g) if case["ragged"] else None
    return {"target": target, "draft": draft, "drafted": drafted, "uniforms": _uniform(g, b, k + 1), "lengths": lengths}


def _inputs(case, seed):
    return {"route": _route_inputs, "int8": _int8_inputs, "verify": _verify_inputs}[case["op"]](_generator(seed), case)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], s["graph"] = case, None
    if own and case["op"] == "int8":
        # the layout in HBM that a program keeps its weights in
        from vibeblade_amd.int8 import Int8QTensor
        s["weights"] = [(Int8QTensor.from_int8(w["codes"], w["scales"]), w["bias"]) for w in s.pop("mats")]
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
    if case["op"] == "route":
        from vibeblade_amd.tensor import route_experts
        return [route_experts(r["logits"], case["topk"], scores=case["scores"], bias=r["bias"], groups=case["groups"],
                              groups_kept=case["kept"], group_score=case["group_score"], renorm=case["renorm"],
                              scale=case["scale"]) for r in s["routers"]]
    if case["op"] == "int8":
        from vibeblade_amd.int8 import int8_gemm, quantize_tokens
        x = quantize_tokens(s["x"]) if case["shared"] else s["x"]
        return [int8_gemm(w, x, bias=bias, out_dtype=DTYPES[case["out"]]) for w, bias in s["weights"]]
    from vibeblade_amd.tensor import verify_draft
    return verify_draft(s["target"], s["drafted"], s["uniforms"], draft=s["draft"], lengths=s["lengths"],
                        temperature=case["temperature"])


# ---- the plain forms ---------------------------------------------------------

def _plain_route(case, z, bias):
    """In 64 bits: which of two experts comes first is decided by scores that may differ in their last bits."""
    z = z.double()
    tokens, experts, groups = z.shape[0], z.shape[1], case["groups"]
    if case["scores"] == "softmax":
        top = z.max(1, keepdim=True).values
        score = torch.exp(z - torch.where(torch.isinf(top), 0.0, top))
        score = score / score.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        score = 1 / (1 + torch.exp(-z))
    value = score if bias is None else score + bias.double()
    value = torch.where(torch.isinf(z), -math.inf, value)
    choice = z if bias is None else value
    if case["kept"] < groups:
        if case["group_score"] == "max":
            of_group = choice.view(tokens, groups, -1).max(2).values
        else:
            two = value.view(tokens, groups, -1).sort(dim=2, descending=True).values[:, :, :2]
            of_group = two[:, :, 0] + torch.where(torch.isinf(two), 0.0, two)[:, :, 1:].sum(2)
        best = of_group.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        kept = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, best, True)
        choice = torch.where(kept.repeat_interleave(experts // groups, 1), choice, -math.inf)
    best = choice.sort(dim=1, descending=True, stable=True)
    ids, named = best.indices[:, :case["topk"]], best.values[:, :case["topk"]] > -math.inf
    w = torch.where(named, score.gather(1, ids), 0.0)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.where(named, ids, -1).to(torch.int32), (case["scale"] * w).float()


def _plain_int8(case, x, w):
    """The quantizing in 64 bits (a value next to the border of two codes), the product in 32."""
    scale = (x.abs().max(1, keepdim=True).values.double() / 127).float().clamp(min=2.0 ** -126)
    codes = torch.round(x.double() / scale.double()).float()
    y = (codes @ w["codes"].float().T) * scale * w["scales"]
    return (y if w["bias"] is None else y + w["bias"]).to(DTYPES[case["out"]])


def _probabilities(z, temperature):
    z = z.double() / temperature
    top = z.max(-1, keepdim=True).values
    e = torch.exp(z - torch.where(torch.isinf(top), 0.0, top))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def _plain_verify(s):
    """In 64 bits: a sum over a whole vocabulary decides which token a random number names."""
    case, drafted, u = s["case"], s["drafted"], s["uniforms"].double()
    b, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    p = _probabilities(s["target"], case["temperature"])
    at = drafted[..., None]
    q = _probabilities(s["draft"], case["temperature"]) if s["draft"] is not None else None
    q_of = q.gather(2, at)[..., 0] if q is not None else torch.ones_like(u[:, :k])
    length = torch.full((b,), k, device=u.device) if s["lengths"] is None else s["lengths"].long()
    place = torch.arange(k, device=u.device)
    taken = (u[:, :k] * q_of < p[:, :k].gather(2, at)[..., 0]) & (place < length[:, None])
    accepted = taken.long().cumprod(1).sum(1)
    row = torch.arange(b, device=u.device)
    r = p[row, accepted]
    refused = (accepted < length)[:, None]
    j = accepted.clamp(max=k - 1)
    if q is not None:
        rest = (r - q[row, j]).clamp(min=0)
    else:
        rest = r.scatter(1, drafted[row, j][:, None], 0.0)
    r = torch.where(refused & (rest.sum(1, keepdim=True) > 0), rest, r)
    c = r.cumsum(1)
    named = ((c > u[:, k:] * c[:, -1:]) & (r > 0)).to(torch.uint8).argmax(1)
    tokens = torch.where(place < accepted[:, None], drafted, -1)
    tokens = torch.cat([tokens, torch.full((b, 1), -1, device=u.device)], 1).scatter(1, accepted[:, None], named[:, None])
    return tokens.to(torch.int32), accepted.to(torch.int32)


def run(state):
    if own:
        if state["graph"] is not None:
            state["graph"].replay()
            return state["out"]
        return _calls(state)
    case = state["case"]
    if case["op"] == "route":
        return [_plain_route(case, r["logits"], r["bias"]) for r in state["routers"]]
    if case["op"] == "int8":
        return [_plain_int8(case, state["x"], w) for w in state["mats"]]
    return _plain_verify(state)


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    if case["op"] == "route":
        tokens, experts = case["tokens"], case["experts"]
        each = tokens * (experts * SIZE[case["x"]] + 8 * case["topk"]) + (4 * experts if case["bias"] else 0)
        return {"bytes": case["layers"] * each, "flops": case["layers"] * 8 * tokens * experts}
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        each = n * (k + 4 + (4 if case["bias"] else 0)) + m * n * SIZE[case["out"]]
        return {"bytes": case["layers"] * each + m * k * SIZE[case["x"]], "flops": case["layers"] * 2 * m * n * k}
    b, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    rows = b * (2 * k + 1 if case["draft"] else k + 1)
    return {"bytes": rows * vocab * SIZE[case["x"]] + b * (20 * k + 12), "flops": 4 * rows * vocab}


# ---- the definitions in float64 ----------------------------------------------------

def _exact_route(case, s):
    out = []
    for r in s["routers"]:
        z = r["logits"].double()
        open_ = z > -math.inf
        score = torch.softmax(z, 1).nan_to_num(0.0) if case["scores"] == "softmax" else torch.sigmoid(z)
        value = score + (0.0 if r["bias"] is None else r["bias"].double())
        choice = torch.where(open_, z if r["bias"] is None else value, -math.inf)
        size = case["experts"] // case["groups"]
        if case["kept"] < case["groups"]:
            parts = []
            for first in range(0, case["experts"], size):
                if case["group_score"] == "max":
                    parts.append(choice[:, first:first + size].amax(1))
                else:
                    v = torch.where(open_, value, -math.inf)[:, first:first + size]
                    two = torch.topk(v, min(2, size), 1).values
                    parts.append(torch.where(two[:, 0] > -math.inf, torch.where(two > -math.inf, two, 0.0).sum(1), -math.inf))
            of_group = torch.stack(parts, 1)
            # a group's place: how many are larger, or equal and before it
            larger = of_group[:, None, :] > of_group[:, :, None]
            before = torch.arange(case["groups"], device=z.device)
            equal = (of_group[:, None, :] == of_group[:, :, None]) & (before[None, :] < before[:, None])
            stays = ((larger | equal).sum(2) < case["kept"]).repeat_interleave(size, 1)
            choice = torch.where(stays, choice, -math.inf)
        ids, w = [], []
        for _ in range(case["topk"]):
            most = choice.amax(1, keepdim=True)
            first = (choice == most).to(torch.uint8).argmax(1, keepdim=True)  # the lowest index of equal ones
            some = most > -math.inf
            ids.append(torch.where(some, first, -1))
            w.append(torch.where(some, score.gather(1, first), 0.0))
            choice = choice.scatter(1, first, -math.inf)
        w = torch.cat(w, 1)
        if case["renorm"]:
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, 0.0)
        out.append((torch.cat(ids, 1).to(torch.int32), w * case["scale"]))
    return out


def _exact_int8(case, s):
    x, out = s["x"].double(), []
    scale = torch.clamp((x.abs().amax(1) / 127).float(), min=2.0 ** -126).double()  # kept in float32
    codes = (x / scale[:, None]).round()
    for w in s["mats"]:
        y = torch.empty((case["m"], case["n"]), dtype=torch.float64, device=x.device)
        for first in range(0, case["n"], 4096):
            part = w["codes"][first:first + 4096].double()
            y[:, first:first + 4096] = codes @ part.T.contiguous()
        y *= w["scales"].double()
        y *= scale[:, None]
        out.append(y if w["bias"] is None else y + w["bias"].double())
    return out


def _exact_verify(case, s):
    u = s["uniforms"].double().tolist()
    drafted = s["drafted"].tolist()
    lengths = [case["drafts"]] * case["seqs"] if s["lengths"] is None else s["lengths"].tolist()
    tokens, accepted = [], []

    def softmax(z):
        return torch.softmax(z.double() / case["temperature"], 0).nan_to_num(0.0)

    for b in range(case["seqs"]):
        out, end = [], None
        for j in range(lengths[b]):
            p, d = softmax(s["target"][b, j]), drafted[b][j]
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[d] = 1.0
            else:
                q = softmax(s["draft"][b, j])
            if u[b][j] * float(q[d]) < float(p[d]):
                out.append(d)
                continue
            end = torch.relu(p - q)
            end = end if float(end.sum()) > 0 else p
            break
        accepted.append(len(out))
        if end is None:
            end = softmax(s["target"][b, len(out)])
        c = torch.cumsum(end, 0)
        at = int(torch.searchsorted(c, (u[b][case["drafts"]] * c[-1]).reshape(1), right=True))
        out.append(min(at, int(torch.nonzero(end)[-1])))
        tokens.append(out + [-1] * (case["drafts"] + 1 - len(out)))
    device = s["target"].device
    return (torch.tensor(tokens, dtype=torch.int32, device=device),
            torch.tensor(accepted, dtype=torch.int32, device=device))


def exact(case, seed):
    return {"route": _exact_route, "int8": _exact_int8, "verify": _exact_verify}[case["op"]](case, _inputs(case, seed))
