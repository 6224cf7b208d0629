"""The choice of experts against its definition, row by row in 64 bits: ids equal; weights
within one f32 rounding (2^-24) and 64-bit noise."""
import math

import pytest
import torch

from tests import _mx4_ref as R
from tilefoundry_amd.routing import Routing

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16


def _check(rule, logits, bias=None):
    w, ids = rule(logits, bias)
    want_w, want_i = R.route(logits, bias, k=rule.top_k, score=rule.score, groups=rule.groups,
                             keep=rule.kept_groups, group_top=rule.group_top,
                             renormalise=rule.renormalise, scale=rule.scale, shared=rule.shared)
    assert w.dtype == F32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), want_i)
    # 2^-24 for the rounding to f32 (subnormals: their half step), 1e-12 for 64-bit sums
    bound = want_w.abs() * (2.0 ** -24 + 1e-12) + 2.0 ** -150
    assert ((w.cpu().double() - want_w).abs() <= bound).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,keep,top,k", [
    (1, 1, 1, 2, 1), (5, 1, 1, 1, 5), (64, 1, 1, 2, 6), (65, 5, 2, 2, 3), (72, 1, 1, 2, 10),
    (256, 8, 4, 2, 8), (256, 64, 3, 2, 9), (130, 13, 12, 1, 40), (512, 16, 1, 2, 32),
    (512, 64, 64, 1, 64), (32, 32, 7, 2, 7)])
def test_route_matches_definition(gpu_device, score, E, groups, keep, top, k):
    g = torch.Generator().manual_seed(E * 7 + k)
    for rows, dtype, biased in [(1, F32, True), (7, BF, False), (130, F32, True), (33, F16, True)]:
        logits = (torch.randn(rows, E, generator=g) * 2).to(dtype).to(gpu_device)
        bias = (torch.randn(E, generator=g) * 0.2).to(gpu_device) if biased else None
        _check(Routing(top_k=k, score=score, groups=groups, kept_groups=keep, group_top=top,
                       renormalise=rows != 7, scale=2.5 if rows == 130 else 1.0,
                       shared=min(2, 64 - k)), logits, bias)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_masks_ties_and_infinities(gpu_device, score):
    """Rows with no expert, one, fewer than k; NaN, infinities, the types' lowest value;
    rows of equal logits; biases that are not finite."""
    E = 24
    g = torch.Generator().manual_seed(5)
    x = torch.randn(12, E, generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 17] = 0.5
    x[3, ::2] = -math.inf
    x[4] = 1.25                                     # all equal
    x[5] = torch.finfo(F32).min
    x[5, 3] = 0.0
    x[6, 4] = x[6, 9] = math.inf
    x[7] = torch.tensor([0.0, 1.0] * 12)
    x[8] = -math.inf
    x[8, 21], x[8, 2] = -800.0, math.nan             # a sigmoid that is zero in 64 bits
    x[9, :20] = math.nan
    x[10] = torch.finfo(F32).max
    logits = x.to(gpu_device)
    bias = torch.randn(E, generator=g) * 0.1
    for b in [None, bias, bias.clone().index_fill_(0, torch.tensor([1, 4]), -math.inf),
              bias.clone().index_fill_(0, torch.tensor([0, 21]), math.nan),
              bias.clone().index_fill_(0, torch.tensor([5]), math.inf)]:
        b = None if b is None else b.to(gpu_device)
        for groups, keep, k in [(1, 1, 6), (6, 2, 3), (4, 3, 18), (24, 5, 5)]:
            for renormalise in (True, False):
                _check(Routing(top_k=k, score=score, groups=groups, kept_groups=keep,
                               renormalise=renormalise, shared=1), logits, b)


def test_route_strides_empty_and_replayed(gpu_device):
    g = torch.Generator().manual_seed(9)
    rule = Routing(top_k=3, score="sigmoid", groups=4, kept_groups=2)
    wide = torch.randn(20, 50, generator=g).to(gpu_device)
    _check(rule, wide[:, 3:43])
    _check(rule, wide[::3, :40])
    _check(rule, torch.randn(40, 6, generator=g).to(gpu_device).t())
    _check(rule, wide[:1, :40].expand(4, 40))
    w, ids = rule(wide[:0, :40])
    assert w.shape == (0, 3) and ids.shape == (0, 3)
    static = wide[:, :40].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = rule(static)
    for i in range(3):
        static.copy_(torch.randn(20, 40, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        ew, ei = rule(static)
        assert torch.equal(w, ew) and torch.equal(ids, ei)


def test_route_of_many_rows(gpu_device):
    logits = torch.randn(5000, 64, generator=torch.Generator().manual_seed(1)).to(gpu_device)
    _check(Routing(top_k=2), logits)
