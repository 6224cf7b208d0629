"""Drafted trees against their definition in 64 bits: masks, depths and paths equal; attention
within one bf16 rounding of the output (2^-8 of its value, half a step of eight bits) and the
error of its operands: a probability is a sum of two bf16 (2^-16 of it), or one where waves share
positions (2^-8: the form says so), scores are f32 sums of
exact products (2^-24 of the sum of their sizes for each of dim additions, at most dim 2^-24
times |q| |k| here), sums over n positions n 2^-24 of the sum of |p v|."""
import ctypes
import math

import pytest
import torch

from tests import _search_ref as R
from tilefoundry_amd import _lib, tree
from tilefoundry_amd._lib import lib

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _parents(g, rows, nodes):
    back = torch.randint(1, 6, (rows, nodes), generator=g)
    p = torch.clamp(torch.arange(nodes) - back, min=-1)
    return p.to(I32)


def _case(seed, rows, nodes, heads, kv_heads, dim, lengths, spare=3, room=0):
    """*room*: pages more that a row's table has place for (-1: none there)."""
    g = _gen(seed)
    width = max(-(-(n + nodes) // 16) for n in lengths) + 1
    pages = rows * width + spare
    perm = torch.randperm(pages, generator=g)[:rows * width]
    table = torch.full((rows, width + room), -1, dtype=I32)
    table[:, :width] = perm.view(rows, width)
    return {"q": torch.randn(rows, nodes, heads, dim, generator=g).to(BF),
            "k_pool": torch.randn(pages, kv_heads, 16, dim, generator=g).to(BF),
            "v_pool": torch.randn(pages, kv_heads, 16, dim, generator=g).to(BF),
            "table": table,
            "lengths": torch.tensor(lengths, dtype=I32),
            "masks": R.words(R.ancestors(_parents(g, rows, nodes))[0], nodes)}


def _form(c, rows=None):
    rows_, nodes, heads, dim = c["q"].shape
    got = (ctypes.c_int32 * 4)()
    lib().tfd_tree_attn_form(rows or rows_, nodes, heads, c["k_pool"].shape[1], dim,
                             c["table"].shape[1], got)
    return tuple(got)


def _bound(c, want, size, scale):
    """See the module docstring."""
    dim, heads = c["q"].shape[3], c["q"].shape[2]
    operand = 2.0 ** -16 if _form(c)[0] else 2.0 ** -8
    n = int(c["lengths"].max()) + c["q"].shape[1]
    qn = c["q"].double().norm(dim=3).max()
    kn = c["k_pool"].double()
    kn = kn[torch.isfinite(kn).all(3)].norm(dim=1).max()
    score = scale * qn * kn * (dim + 8) * 2.0 ** -24 + 2.0 ** -22     # and exp2's argument
    return want.abs() * 2.0 ** -8 + size * (2 * score + operand + (n + 8) * 2.0 ** -24) + 1e-30


def _check(c, dev, counts=None, scale=None, **kw):
    d = {k: v.to(dev) for k, v in c.items()}
    got = tree.attention(**d, counts=None if counts is None else counts.to(dev), scale=scale,
                         **kw)
    want, size = R.attention(**c, counts=counts, scale=scale)
    there = torch.ones(got.shape[:2], dtype=torch.bool) if counts is None else \
        torch.arange(got.shape[1]) < counts.unsqueeze(1)
    got, want, size = got.cpu().double()[there], want[there], size[there]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    near = (got - want).abs() <= _bound(c, want, size, scale or c["q"].shape[3] ** -0.5)
    same = got == want                               # infinities
    assert (near | same)[ok].all(), (got - want).abs()[ok].max()


@pytest.mark.parametrize("rows,nodes", [(1, 1), (3, 7), (2, 64), (2, 65), (1, 255), (2, 256)])
def test_ancestors(gpu_device, rows, nodes):
    p = _parents(_gen(nodes), rows, nodes)
    p[0] = torch.arange(nodes) - 1                   # a chain
    for counts in (None, torch.tensor([nodes // 2, nodes, 0][:rows], dtype=I32)):
        masks, depths = tree.ancestors(p.to(gpu_device),
                                       None if counts is None else counts.to(gpu_device))
        sets, want = R.ancestors(p, counts)
        assert torch.equal(masks.cpu(), R.words(sets, nodes))
        assert depths.cpu().tolist() == want


def test_ancestors_of_parents_out_of_range(gpu_device):
    p = torch.tensor([[-1, 0, 5, 2, -2, 3]], dtype=I32)
    err = torch.zeros(1, dtype=I32, device=gpu_device)
    masks, depths = tree.ancestors(p.to(gpu_device), err=err)
    sets, want = R.ancestors(p)
    assert torch.equal(masks.cpu(), R.words(sets, 6)) and depths.cpu().tolist() == want
    assert err.item() == _lib.ERR_ROW_RANGE


@pytest.mark.parametrize("rows,nodes", [(1, 1), (5, 9), (3, 64), (2, 200), (2, 256)])
def test_accept(gpu_device, rows, nodes):
    g = _gen(nodes + 1)
    parents = _parents(g, rows, nodes)
    tokens = torch.randint(0, 3, (rows, nodes), generator=g, dtype=I32)
    picks = torch.randint(0, 3, (rows, nodes), generator=g, dtype=I32)
    if rows > 1:                                     # a chain that is accepted whole
        parents[1] = torch.arange(nodes) - 1
        picks[1, :-1] = tokens[1, 1:]
    for counts in (None, torch.tensor([nodes, nodes - 1, 0, 1, nodes][:rows], dtype=I32)):
        d = [x.to(gpu_device) for x in (tokens, parents, picks)]
        got = tree.accept(*d, None if counts is None else counts.to(gpu_device))
        for a, b in zip(got, R.accept(tokens, parents, picks, counts)):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("rows,nodes,heads,kv_heads,dim,lengths", [
    (1, 1, 1, 1, 64, [0]), (1, 1, 2, 1, 128, [1]), (2, 3, 4, 2, 256, [0, 17]),
    (1, 16, 16, 8, 128, [700]), (3, 7, 4, 2, 128, [15, 16, 33]), (2, 8, 4, 2, 64, [31, 32]),
    (2, 33, 8, 2, 128, [5, 190]), (1, 64, 4, 1, 128, [100]), (1, 65, 2, 1, 64, [63]),
    (2, 13, 16, 2, 256, [1, 301]), (1, 130, 6, 3, 128, [47]), (1, 256, 2, 2, 64, [20]),
    (4, 5, 14, 2, 64, [0, 3, 1000, 64]), (1, 20, 5, 1, 128, [2100])])
def test_attention(gpu_device, rows, nodes, heads, kv_heads, dim, lengths):
    c = _case(rows * 100 + nodes, rows, nodes, heads, kv_heads, dim, lengths)
    _check(c, gpu_device)


FORMS = [  # (rows, nodes, heads, kv heads, dim, room), form: how such calls run
    ((1, 7, 4, 2, 64, 9), (1, 16, 1, 1)), ((2, 20, 4, 2, 128, 9), (1, 12, 3, 1)),
    ((1, 13, 8, 2, 256, 9), (1, 8, 4, 1)),
    ((1, 31, 8, 2, 64, 90), (1, 16, 8, 3)), ((2, 11, 4, 2, 128, 400), (1, 12, 2, 17)),
    ((2, 9, 8, 2, 256, 60), (1, 8, 3, 4)),
    ((3, 7, 4, 2, 64, 100), (1, 4, 1, 13)), ((3, 7, 4, 2, 128, 100), (1, 4, 1, 13)),
    ((3, 4, 8, 2, 256, 100), (1, 4, 1, 13)), ((64, 2, 16, 8, 64, 400), (1, 4, 1, 1)),
    ((6, 16, 16, 8, 64, 400), (2, 4, 1, 5)), ((6, 16, 16, 8, 128, 400), (2, 4, 1, 5)),
    ((36, 11, 16, 8, 64, 400), (2, 4, 1, 1)), ((36, 31, 16, 8, 128, 40), (2, 4, 2, 1)),
    ((2, 21, 8, 2, 64, 400), (0, 4, 1, 25)), ((2, 21, 8, 2, 128, 400), (0, 8, 1, 25)),
    ((2, 13, 8, 2, 256, 400), (0, 8, 1, 25)), ((1, 61, 8, 2, 128, 400), (0, 8, 1, 25)),
    ((1, 61, 16, 2, 64, 400), (0, 8, 2, 25)), ((1, 39, 16, 2, 256, 400), (0, 8, 2, 25)),
    ((33, 33, 16, 8, 128, 400), (0, 4, 1, 1)), ((33, 66, 16, 8, 64, 9), (0, 8, 1, 1)),
    ((33, 10, 16, 8, 256, 100), (0, 8, 1, 1))]


@pytest.mark.parametrize("shape,form", FORMS)
def test_attention_forms(gpu_device, shape, form):
    """Every way a call may run: with its rows' tables far longer than the rows; drafted values
    that are not finite, absent nodes."""
    rows, nodes, heads, kv_heads, dim, room = shape
    lengths = [(71 * b + 13) % 210 if rows > 8 or b else 333 for b in range(rows)]
    c = _case(sum(shape), rows, nodes, heads, kv_heads, dim, lengths, room=room)
    got = _form(c)
    assert got[:3] == form[:3] and (got[3] > 1) == (form[3] > 1), got
    if rows > 8:                                     # the reference takes its time
        few = torch.tensor([0, 7, rows - 1])
        d = {k: v.to(gpu_device) for k, v in c.items()}
        out = tree.attention(**d).cpu()[few]
        part = {**c, **{k: c[k][few] for k in ("q", "table", "lengths", "masks")}}
        want, size = R.attention(**part)
        assert ((out.double() - want).abs() <= _bound(c, want, size, dim ** -0.5)).all()
        return
    _check(c, gpu_device)
    counts = torch.tensor(([nodes - 1, 0, nodes] * 3)[:rows], dtype=I32)
    c["masks"][0, nodes // 2:] &= ~2
    at = 333 + 1                                     # node 1's value
    c["v_pool"][c["table"][0, at // 16].long(), 0, at % 16, 5] = math.inf
    c["v_pool"][c["table"][0, at // 16].long(), 0, at % 16, dim - 1] = math.nan
    _check(c, gpu_device, counts=counts)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_counts_scale_and_any_mask(gpu_device, dim):
    """Rows of fewer nodes (none, one), masks of any bits, a scale of one's own."""
    c = _case(dim, 4, 21, 6, 2, dim, [0, 40, 200, 7])
    g = _gen(dim + 1)
    c["masks"] = torch.randint(0, 1 << 21, c["masks"].shape, generator=g)
    c["masks"][0, 3] = 0                             # no position, no node: zeros
    c["masks"][2, 5] = 0                             # its context alone
    counts = torch.tensor([9, 0, 21, 1], dtype=I32)
    _check(c, gpu_device, counts=counts, scale=0.21)


def test_attention_leaves_absent_nodes_alone(gpu_device):
    c = _case(3, 2, 6, 4, 2, 128, [50, 3])
    d = {k: v.to(gpu_device) for k, v in c.items()}
    counts = torch.tensor([2, 0], dtype=I32, device=gpu_device)
    whole = tree.attention(**d)
    some = tree.attention(**d, counts=counts)
    del whole
    c["masks"][0, 0] = 1
    want, _ = R.attention(**c, counts=counts.cpu())
    assert some.shape == (2, 6, 4, 128)
    assert torch.allclose(some[0, :2].cpu().double(), want[0, :2], atol=0.03)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_leaves_out_what_a_node_does_not_see(gpu_device, bad):
    """Values and keys that are not finite: behind the last position, in pages that no row
    has, in nodes that others do not see."""
    c = _case(11, 2, 12, 4, 2, 128, [37, 5])
    n = [49, 17]
    for b in range(2):
        for pos in range(n[b], c["table"].shape[1] * 16):
            for pool in ("k_pool", "v_pool"):
                c[pool][c["table"][b, pos // 16].long(), :, pos % 16] = bad
    used = set(c["table"].flatten().tolist())
    for page in range(c["k_pool"].shape[0]):
        if page not in used:
            c["k_pool"][page] = c["v_pool"][page] = bad
    # node 4's value is not finite: those that see it are not either, the others are
    c["masks"][:, 7:] &= ~(1 << 4)
    pos = 37 + 4
    c["v_pool"][c["table"][0, pos // 16].long(), 1, pos % 16, 3:9] = bad
    _check(c, gpu_device)
    # a key of it: seen, a score that is not finite
    c = _case(12, 1, 12, 4, 2, 64, [37])
    c["masks"][:, 7:] &= ~(1 << 4)
    c["k_pool"][c["table"][0, pos // 16].long(), 0, pos % 16] = math.nan
    _check(c, gpu_device)


def test_attention_large_scores_and_far_maxima(gpu_device):
    """Scores of some hundreds, the largest at the first, a middle and the last position."""
    for at in (0, 700, 1399):
        c = _case(at, 1, 3, 2, 1, 128, [1400])
        c["q"] *= 8
        page = c["table"][0, at // 16].long()
        c["k_pool"][page, :, at % 16] = c["q"][0, 0, 0] * 0.5
        _check(c, gpu_device)


def test_attention_strides_streams_and_graphs(gpu_device):
    """Queries inside a wider projection, tensors on a side stream, a graph replayed with other
    lengths."""
    c = _case(5, 3, 5, 4, 2, 128, [20, 100, 64])
    d = {k: v.to(gpu_device) for k, v in c.items()}
    want = tree.attention(**d)
    wide = torch.zeros(3, 5, 9, 128, dtype=BF, device=gpu_device)
    wide[:, :, 2:6] = d["q"]
    odd = torch.zeros(3 * 5 * 4 * 128 + 3, dtype=BF, device=gpu_device)[3:].view(3, 5, 4, 128)
    odd.copy_(d["q"])
    turned = d["q"].permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    for q in (wide[:, :, 2:6], odd, turned):
        assert torch.equal(tree.attention(**{**d, "q": q}), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tree.attention(**d)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree.attention(**d)
    for lengths in ([20, 100, 64], [0, 3, 90], [99, 1, 1], [20, 100, 64]):
        d["lengths"].copy_(torch.tensor(lengths, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, tree.attention(**d))


def test_attention_flags_what_is_out_of_range(gpu_device):
    c = _case(6, 2, 4, 4, 2, 64, [30, 9])
    d = {k: v.to(gpu_device) for k, v in c.items()}
    want = tree.attention(**d)
    err = torch.zeros(1, dtype=I32, device=gpu_device)
    d["lengths"][1] = 16 * c["table"].shape[1] - 3
    got = tree.attention(**d, err=err)
    assert err.item() == _lib.ERR_POS_RANGE
    assert torch.equal(got[0], want[0]) and not got[1].any()
    err.zero_()
    d["lengths"][1] = 9
    d["table"][1, 0] = c["k_pool"].shape[0]
    got = tree.attention(**d, err=err)
    assert err.item() == _lib.ERR_PAGE_RANGE and torch.equal(got[0], want[0])


def test_attention_offsets_past_32_bits(gpu_device):
    """Pages whose elements lie past 2^31 of their pool."""
    rows, nodes, kv_heads, dim = 1, 3, 8, 256
    pages = (1 << 31) // (kv_heads * 16 * dim) + 40
    k = torch.zeros(pages, kv_heads, 16, dim, dtype=BF, device=gpu_device)
    v = torch.zeros(pages, kv_heads, 16, dim, dtype=BF, device=gpu_device)
    g = _gen(9)
    far = torch.arange(pages - 6, pages)
    small = torch.randn(2, 6, kv_heads, 16, dim, generator=g).to(BF)
    k[far.to(gpu_device)] = small[0].to(gpu_device)
    v[far.to(gpu_device)] = small[1].to(gpu_device)
    q = torch.randn(rows, nodes, 16, dim, generator=g).to(BF)
    masks = R.words(R.ancestors(torch.tensor([[-1, 0, 0]]))[0], nodes)
    table = far.flip(0).view(1, 6).to(I32)
    lengths = torch.tensor([70], dtype=I32)
    got = tree.attention(q.to(gpu_device), k, v, table.to(gpu_device), lengths.to(gpu_device),
                         masks.to(gpu_device))
    c = {"q": q, "k_pool": small[0], "v_pool": small[1], "table": table - (pages - 6),
         "lengths": lengths, "masks": masks}
    want, size = R.attention(**c)
    assert ((got.cpu().double() - want).abs() <= _bound(c, want, size, 1 / 16)).all()


def test_empty_calls(gpu_device):
    z = torch.zeros(0, 4, dtype=I32, device=gpu_device)
    assert tree.ancestors(z)[0].shape == (0, 4, 1)
    assert tree.accept(z, z, z)[0].shape == (0, 4)
    pool = torch.zeros(2, 1, 16, 64, dtype=BF, device=gpu_device)
    out = tree.attention(torch.zeros(0, 4, 2, 64, dtype=BF, device=gpu_device), pool, pool,
                         torch.zeros(0, 3, dtype=I32, device=gpu_device),
                         torch.zeros(0, dtype=I32, device=gpu_device),
                         torch.zeros(0, 4, 1, dtype=torch.int64, device=gpu_device))
    assert out.shape == (0, 4, 2, 64)
