"""Microscaled tensors, the experts' choice and their products from their definitions, in
64 bits on the CPU, row by row where that is plainest."""
import math

import torch

F64 = torch.float64
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                    dtype=F64)


def values(codes, scales):
    """The f64 values of codes [..., K/2] and scales [..., K/32]; scale 255 is NaN."""
    codes, scales = codes.cpu(), scales.cpu()
    v = torch.stack((GRID[(codes & 15).long()], GRID[(codes >> 4).long()]), -1).flatten(-2)
    s = torch.ldexp(torch.ones((), dtype=F64), scales.to(torch.int32) - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def quantise(x):
    """(codes, scales) of rows [..., K]: block by block, the nearest grid point by
    distance, ties to the even code."""
    x = x.cpu().to(F64)
    b = x.reshape(-1, 32)
    codes = torch.zeros(b.shape, dtype=torch.uint8)
    scales = torch.zeros(b.shape[0], dtype=torch.uint8)
    for i, row in enumerate(b):
        if not torch.isfinite(row).all():
            scales[i] = 255
            continue
        top = float(row.abs().max())
        e = -127 if top == 0 else min(max(math.frexp(top)[1] - 1 - 2, -127), 125)
        scales[i] = e + 127
        v = torch.ldexp(row, torch.tensor(-e)).abs().clamp(max=6.0)
        far = (v.unsqueeze(1) - GRID[:8]).abs()
        near = far.min(1, keepdim=True).values
        hit = far == near                      # one code, or two neighbours at a tie
        first = hit.to(torch.int8).argmax(1)
        two = hit.sum(1) == 2
        code = torch.where(two & (first % 2 == 1), first + 1, first)
        codes[i] = code.to(torch.uint8) + 8 * torch.signbit(row).to(torch.uint8)
    codes = codes.reshape(x.shape)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4),
            scales.reshape(*x.shape[:-1], x.shape[-1] // 32))


def route(logits, bias, *, k, score, groups=1, keep=1, group_top=2, renormalise=True,
          scale=1.0, shared=0):
    """(weights f64, ids) row by row."""
    rows, E = logits.shape
    per = E // groups
    out_w, out_i = [], []
    bias = [0.0] * E if bias is None else [float(b) for b in bias.cpu()]
    for row in logits.cpu().to(F64).tolist():
        row = [-math.inf if v != v else v for v in row]
        top = max(row)
        if score == "sigmoid":
            s = [0.0 if v < -700 else 1 / (1 + math.exp(-v)) for v in row]
        else:
            p = [0.0 if v == -math.inf else 1.0 if v == top else math.exp(v - top) for v in row]
            s = [v / sum(p) if sum(p) else 0.0 for v in p]
        c = [-math.inf if row[e] == -math.inf or bias[e] != bias[e] else s[e] + bias[e]
             for e in range(E)]

        def rank(g):
            best = sorted((v for v in c[g * per:(g + 1) * per] if v > -math.inf), reverse=True)
            return -sum(best[:group_top]) if best else math.inf

        kept = sorted(range(groups), key=lambda g: (rank(g), g))[:keep]
        may = [e for g in kept for e in range(g * per, (g + 1) * per) if c[e] > -math.inf]
        picks = sorted(may, key=lambda e: (-c[e], e))[:k]
        total = sum(s[e] for e in picks)
        w = [s[e] * scale if not renormalise else s[e] / total * scale if total else 0.0
             for e in picks]
        none = k - len(picks)
        out_w.append(w + [0.0] * none + [1.0] * shared)
        out_i.append(picks + [-1] * none + list(range(E, E + shared)))
    n = k + shared
    return (torch.tensor(out_w, dtype=F64).reshape(rows, n),
            torch.tensor(out_i, dtype=torch.int32).reshape(rows, n))


def experts(x, ids, weights, gate, up, down, hidden_dtype=torch.bfloat16):
    """sum over slots of weight * down(round(silu(gate x) * (up x))), f64 otherwise; the
    hidden values rounded as the kernels round them.  gate, up, down: f64 [E][...] values."""
    x, weights = x.cpu().to(F64), weights.cpu().to(F64)
    out = torch.zeros(x.shape[0], down.shape[1], dtype=F64)
    for r, row in enumerate(ids.cpu().tolist()):
        for j, e in enumerate(row):
            if not 0 <= e < gate.shape[0]:
                continue
            a = gate[e] @ x[r]
            h = a / (1 + torch.exp(-a)) * (up[e] @ x[r])
            if hidden_dtype is not None:
                h = h.to(hidden_dtype).to(F64)
            out[r] += weights[r, j] * (down[e] @ h)
    return out
