"""Operators of 4-bit mixture-of-experts serving, as measurable cases.

* ``quantise``: rows to microscaled 4-bit floating point (e2m1 elements, one power-of-two
  scale for each 32 along a row) and back to the values it stands for;
* ``linear``: a projection by microscaled 4-bit weights, of bf16 rows or (``both``) of rows
  that the call quantises too;
* ``route``: the choice of experts for each row;
* ``experts``: the chosen experts' gated products, weighted and summed.

Sizes are those of this repository's models: Qwen3-1.7B (hidden 2,048, 6,144 inner columns),
Qwen3.5 (hidden 2,048, 256 experts of 512, 8 a token) and Granite-4.0-H (hidden 4,096, 72
experts of 768, 10 a token).
"""
from __future__ import annotations

import math

import torch

own = False

BF, F32, F64, I32, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.uint8
DEV = "cuda:0"
TYPES = {"bf16": BF, "f32": F32, "f16": torch.float16}
BLOCK = 32                        # elements that share a scale


# --------------------------------------------------------------------- the cases
def listed():
    return [
        # a step's activations before a product of two 4-bit operands
        {"name": "quantise 16 rows", "kind": "quantise", "rows": 16, "K": 4096, "type": "bf16"},
        # a Qwen3 gate/up matrix at load time, from 32-bit weights
        {"name": "quantise weights", "kind": "quantise", "rows": 12288, "K": 2048,
         "type": "f32"},
        # gate/up of one sequence's decode step
        {"name": "linear 1 row", "kind": "linear", "rows": 1, "K": 2048, "N": 12288,
         "both": False, "out": "bf16"},
        # down projection of a batch that is no multiple of a tile
        {"name": "linear 19 rows", "kind": "linear", "rows": 19, "K": 6144, "N": 2048,
         "both": False, "out": "f32"},
        # gate/up of a 4,001-token prompt
        {"name": "linear prompt", "kind": "linear", "rows": 4001, "K": 2048, "N": 12288,
         "both": False, "out": "bf16"},
        # Granite's in-projection of a prompt pass, activations in 4 bits too
        {"name": "linear prompt both", "kind": "linear", "rows": 4001, "K": 4096, "N": 8512,
         "both": True, "out": "bf16"},
        # the router of one token: softmax over 256, top 8, renormalised
        {"name": "route 1 row", "kind": "route", "rows": 1, "experts": 256, "k": 8, "groups": 1,
         "keep": 1, "score": "softmax", "bias": False, "type": "f32"},
        # the router of a prompt: sigmoid scores, a balancing bias, 4 of 8 groups
        {"name": "route prompt", "kind": "route", "rows": 4001, "experts": 256, "k": 8,
         "groups": 8, "keep": 4, "score": "sigmoid", "bias": True, "type": "f32"},
        # one token of a Qwen3.5 layer
        {"name": "experts 1 row", "kind": "experts", "rows": 1, "experts": 256, "k": 8,
         "H": 2048, "I": 512},
        # a Granite layer's decode step of eight sequences
        {"name": "experts 8 rows", "kind": "experts", "rows": 8, "experts": 72, "k": 10,
         "H": 4096, "I": 768},
        # a Qwen3.5 prompt of 250 tokens: about eight rows an expert
        {"name": "experts 250 rows", "kind": "experts", "rows": 250, "experts": 256, "k": 8,
         "H": 2048, "I": 512},
        # a Granite prompt pass of 1,024 rows
        {"name": "experts 1024 rows", "kind": "experts", "rows": 1024, "experts": 72, "k": 10,
         "H": 4096, "I": 768},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "route", "experts", "experts"])
    if kind == "quantise":
        K = BLOCK * _spread(rng, 1, 256)
        return {"kind": kind, "rows": _spread(rng, 1, min(12288, 25_000_000 // K)), "K": K,
                "type": rng.choice(["bf16", "f32", "f16"])}
    if kind == "linear":
        K = BLOCK * _spread(rng, 2, 192)
        N = _spread(rng, 33, 12288)
        rows = _spread(rng, 1, max(1, min(4096, 100_000_000_000 // (K * N))))
        return {"kind": kind, "rows": rows, "K": K, "N": N, "both": rng.random() < 0.4,
                "out": rng.choice(["bf16", "f32"])}
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.randint(max(4, 16 // groups), 256 // groups)
        keep = rng.randint(max(1, groups // 2), groups)
        return {"kind": kind, "rows": _spread(rng, 1, 4096), "experts": experts,
                "k": rng.randint(1, min(12, keep * (experts // groups))), "groups": groups,
                "keep": keep, "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.6, "type": rng.choice(["f32", "bf16"])}
    H, I = BLOCK * rng.randint(8, 128), BLOCK * rng.randint(4, 24)
    experts = rng.randint(8, min(128, 2048 * 512 * 256 // (H * I)))
    k = rng.randint(1, min(10, experts))
    return {"kind": kind, "rows": _spread(rng, 1, 1024), "experts": experts, "k": k, "H": H,
            "I": I}


# ------------------------------------------------------------------ drawn inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rn(g, *shape, s=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device=DEV) * s).to(dtype)


def _weights(g, *shape):
    """Codes and scales of N(0, 0.02) weights."""
    return _to_codes(_rn(g, *shape, s=0.02))


def _inputs(case, seed):
    g = _gen(seed)
    kind, rows = case["kind"], case["rows"]
    if kind == "quantise":
        # activations have outlier channels, weights do not
        x = _rn(g, rows, case["K"], s=0.02 if case["type"] == "f32" else 1.0)
        if case["type"] != "f32":
            x = x * (1 + 20 * (torch.rand(case["K"], generator=g, device=DEV) < 0.01))
        return {"x": x.to(TYPES[case["type"]])}
    if kind == "linear":
        codes, scales = _weights(g, case["N"], case["K"])
        return {"x": _rn(g, rows, case["K"], dtype=BF), "codes": codes, "scales": scales}
    if kind == "route":
        logits = _rn(g, rows, case["experts"], s=1.5, dtype=TYPES[case["type"]])
        bias = _rn(g, case["experts"], s=0.1) if case["bias"] else None
        return {"logits": logits, "bias": bias}
    E, H, I, k = case["experts"], case["H"], case["I"], case["k"]
    # some experts are picked more often than others
    like = _rn(g, 1, E, s=0.7) + _rn(g, rows, E)
    top = torch.topk(like, k, dim=1)
    return {"x": _rn(g, rows, H, dtype=BF), "ids": top.indices.to(I32),
            "weights": torch.softmax(top.values, 1),
            "gate": _weights(g, E, I, H), "up": _weights(g, E, I, H),
            "down": _weights(g, E, H, I)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:                       # the handles that a serving program keeps
        from tilefoundry_amd import mx4, routing

        if case["kind"] == "linear":
            s["handle"] = mx4.Linear(mx4.Mx4(s["codes"], s["scales"]))
        elif case["kind"] == "route":
            s["handle"] = routing.Routing(
                top_k=case["k"], score=case["score"], groups=case["groups"],
                kept_groups=case["keep"])
        elif case["kind"] == "experts":
            s["handle"] = mx4.Experts(mx4.Mx4(*s["gate"]), mx4.Mx4(*s["up"]),
                                      mx4.Mx4(*s["down"]))
    return s


# ------------------------------------------------------------------ plain forms
def _to_codes(x):
    """Codes (two to a byte, the even element low) and scale bytes of rows of finite values."""
    b = x.to(F32).unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.clamp(torch.frexp(top).exponent - 3, -127, 125)
    e = torch.where(top == 0, torch.full_like(e, -127), e)
    v = torch.ldexp(b, -e).abs()
    # the eight magnitudes' midpoints; a tie goes to the even code
    q = ((v > 0.25).to(U8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) +
         (v > 5.0))
    q = (q + 8 * torch.signbit(b)).to(U8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), (e.squeeze(-1) + 127).to(U8)


def _from_codes(codes, scales):
    """The 32-bit values that codes and scales stand for."""
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    grid = torch.cat((half, -half))
    v = torch.stack((grid[(codes & 15).to(I32)], grid[(codes >> 4).to(I32)]), -1).flatten(-2)
    return torch.ldexp(v.unflatten(-1, (-1, BLOCK)),
                       scales.to(I32).unsqueeze(-1) - 127).flatten(-2)


def _route(case, logits, bias):
    E, G, k = case["experts"], case["groups"], case["k"]
    l64 = logits.to(F64)
    s = torch.sigmoid(l64) if case["score"] == "sigmoid" else torch.softmax(l64, 1)
    c = s if bias is None else s + bias.to(F64)
    best = torch.sort(c.unflatten(1, (G, E // G)), dim=2, descending=True).values[:, :, :2].sum(2)
    kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["keep"]]
    mask = torch.zeros_like(best).scatter(1, kept, 1.0).repeat_interleave(E // G, 1)
    c = torch.where(mask > 0, c, torch.full_like(c, -math.inf))
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    return (w / w.sum(1, keepdim=True)).to(F32), ids.to(I32)


def _experts(case, x, ids, weights, gate, up, down):
    E, k, rows = case["experts"], case["k"], case["rows"]
    flat, n = ids.flatten().long(), rows * k
    x = x.to(F32)
    if n <= E:                    # a copy of the expert for each entry
        xe = x.repeat_interleave(k, 0).unsqueeze(2)
        a = _from_codes(gate[0][flat], gate[1][flat]) @ xe
        b = _from_codes(up[0][flat], up[1][flat]) @ xe
        y = (_from_codes(down[0][flat], down[1][flat]) @ (a * torch.sigmoid(a) * b)).squeeze(2)
    else:                         # entries in order of their expert, each expert's padded
        order = torch.sort(flat, stable=True).indices
        e = flat[order]
        count = torch.bincount(flat, minlength=E)
        most = int(count.max())
        place = torch.arange(n, device=DEV) - (torch.cumsum(count, 0) - count)[e]
        xe = torch.zeros(E, x.shape[1], most, device=DEV)
        xe[e, :, place] = x[order // k]
        a = _from_codes(*gate) @ xe
        b = _from_codes(*up) @ xe
        d = _from_codes(*down) @ (a * torch.sigmoid(a) * b)
        y = torch.empty(n, x.shape[1], device=DEV)
        y[order] = d[e, :, place]
    return (y.unflatten(0, (rows, k)) * weights.unsqueeze(2)).sum(1).to(BF)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from tilefoundry_amd import mx4

        if kind == "quantise":
            return mx4.quantise(state["x"]).dequantise(BF)
        if kind == "linear":
            x = mx4.quantise(state["x"]) if case["both"] else state["x"]
            return state["handle"](x, dtype=TYPES[case["out"]])
        if kind == "route":
            return state["handle"](state["logits"], state["bias"])
        return state["handle"](state["x"], state["ids"], state["weights"])
    if kind == "quantise":
        return _from_codes(*_to_codes(state["x"])).to(BF)
    if kind == "linear":
        x = _from_codes(*_to_codes(state["x"])) if case["both"] else state["x"].to(F32)
        return (x @ _from_codes(state["codes"], state["scales"]).t()).to(TYPES[case["out"]])
    if kind == "route":
        return _route(case, state["logits"], state["bias"])
    return _experts(case, state["x"], state["ids"], state["weights"], state["gate"],
                    state["up"], state["down"])


# ------------------------------------------------------------- work and exactness
def work(case):
    kind, rows = case["kind"], case["rows"]
    if kind == "quantise":
        n = rows * case["K"]
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + 2 * n, "flops": 4 * n}
    if kind == "linear":
        K, N = case["K"], case["N"]
        return {"bytes": N * K * 17 // 32 + 2 * rows * K +
                rows * N * (4 if case["out"] == "f32" else 2), "flops": 2 * rows * N * K}
    if kind == "route":
        n = rows * case["experts"]
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + 8 * rows * case["k"],
                "flops": 40 * n}
    E, H, I, n = case["experts"], case["H"], case["I"], rows * case["k"]
    # the experts that n picks touch, were they even
    touched = E * (1 - (1 - case["k"] / E) ** rows)
    return {"bytes": int(touched * 3 * H * I * 17 / 32) + 4 * rows * H + 8 * n,
            "flops": 6 * n * H * I}


def _value64(codes, scales):
    """The definition in 64 bits: sign, two exponent bits, one mantissa bit; 2^(scale - 127)."""
    n = torch.stack((codes.remainder(16), codes.div(16, rounding_mode="floor")), -1)
    n = n.flatten(-2).to(torch.int64)
    exponent, mantissa = n.div(2, rounding_mode="floor").remainder(4), n.remainder(2)
    size = torch.where(exponent > 0, (1 + 0.5 * mantissa) * torch.pow(2.0, exponent.to(F64) - 1),
                       0.5 * mantissa.to(F64))
    scale = torch.pow(torch.full((), 2.0, dtype=F64, device=codes.device), scales.to(F64) - 127)
    return torch.where(n >= 8, -size, size) * scale.repeat_interleave(BLOCK, -1)


def _quantised64(x):
    """x's nearest microscaled values: the grid's nearest point, ties to the even code."""
    x = x.to(F64)
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -140)))
    # log2 of a number just under a power of two may round up to it
    e = torch.where(torch.pow(2.0, e) > top, e - 1, e)
    scale = torch.pow(2.0, torch.clamp(e - 2, -127, 125))
    v = (b / scale).abs().clamp(max=6.0)
    # between two grid points a step apart, half-even rounding of v / step
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0)).to(F64)
    q = torch.round(v / step) * step
    return (torch.sign(b) * q * scale).reshape(x.shape)


def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "quantise":
        return _quantised64(s["x"])
    if kind == "linear":
        x = _quantised64(s["x"]) if case["both"] else s["x"].to(F64)
        return torch.matmul(x, _value64(s["codes"], s["scales"]).transpose(0, 1).contiguous())
    if kind == "route":
        E, G, k = case["experts"], case["groups"], case["k"]
        l64 = s["logits"].to(F64).cpu()
        if case["score"] == "sigmoid":
            p = 1 / (1 + torch.exp(-l64))
        else:
            p = torch.exp(l64 - l64.max(1, keepdim=True).values)
            p = p / p.sum(1, keepdim=True)
        choice = p if s["bias"] is None else p + s["bias"].to(F64).cpu()
        weights, ids = [], []
        for c, q in zip(choice.tolist(), p.tolist()):
            per = E // G
            rank = sorted(range(G), key=lambda j: (-sum(sorted(c[j * per:(j + 1) * per])[-2:]), j))
            may = sorted((i for j in rank[:case["keep"]] for i in range(j * per, (j + 1) * per)),
                         key=lambda i: (-c[i], i))[:k]
            total = sum(q[i] for i in may)
            ids.append(may)
            weights.append([q[i] / total for i in may])
        return (torch.tensor(weights, dtype=F64, device=DEV),
                torch.tensor(ids, dtype=I32, device=DEV))
    out = torch.zeros(case["rows"], case["H"], dtype=F64, device=DEV)
    x = s["x"].to(F64)
    for e in range(case["experts"]):
        row, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not row.numel():
            continue
        g, u, d = (_value64(s[m][0][e], s[m][1][e]) for m in ("gate", "up", "down"))
        a = torch.matmul(x[row], g.transpose(0, 1).contiguous())
        h = a / (1 + torch.exp(-a)) * torch.matmul(x[row], u.transpose(0, 1).contiguous())
        y = torch.matmul(h, d.transpose(0, 1).contiguous())
        out.index_add_(0, row, y * s["weights"][row, slot].to(F64).unsqueeze(1))
    return out
