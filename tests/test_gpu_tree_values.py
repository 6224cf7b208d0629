"""Tree attention where its values, pages and lengths are unusual, by every way a call may run,
against the definition in 64 bits.

The bound is that of a probability as a sum of two bf16 in every form: what two of them leave out
is 2^-8 of the second, itself 2^-8 of the first (half steps of eight bits), so 2^-16 of it; one
bf16 rounding of the output, 2^-8 of its value; scores are f32 sums of exact products, dim 2^-24
times |q| |k|, and the exponential's argument 2^-22; sums over n positions n 2^-24 of the sum of
|p v|."""
import ctypes
import math

import pytest
import torch

from tests import _search_ref as R
from tests.test_gpu_tree import BF, FORMS, I32, _case, _form, _gen
from tilefoundry_amd import _lib, tree
from tilefoundry_amd._lib import lib, ptr

pytestmark = pytest.mark.gpu

MANY = [f for f in FORMS if f[1][0] == 0]


def _lengths(rows):
    return [(71 * b + 13) % 210 if rows > 8 or b else 333 for b in range(rows)]


def _shape(shape, **kw):
    rows, nodes, heads, kv_heads, dim, room = shape
    return _case(sum(shape), rows, nodes, heads, kv_heads, dim, _lengths(rows), room=room, **kw)


def _place(c, b, pos):
    return c["table"][b, pos // 16].long(), pos % 16


def _node(c, b, t):
    """(f64 output of node t of row b [heads, dim], the sum of |p v|); a position whose page is
    none of the pool's is left out."""
    pages, kv_heads = c["k_pool"].shape[:2]
    nodes, heads, dim = c["q"].shape[1:]
    L = int(c["lengths"][b])
    see = [j for j in range(nodes) if (int(c["masks"][b, t, j // 64]) >> (j % 64)) & 1]
    at = torch.cat((torch.arange(L), torch.tensor(see, dtype=torch.int64) + L))
    page = c["table"][b, at // 16].long()
    held = (page >= 0) & (page < pages)
    page, at = page[held], at[held]
    if not len(at):
        return torch.zeros(heads, dim).double(), torch.zeros(heads, dim).double()
    k, v = (c[p][page, :, at % 16].double() for p in ("k_pool", "v_pool"))
    out, size = (torch.empty(heads, dim, dtype=torch.float64) for _ in range(2))
    for h in range(heads):
        g = h // (heads // kv_heads)
        p = torch.softmax(dim ** -0.5 * (k[:, g] @ c["q"][b, t, h].double()), 0).unsqueeze(1)
        out[h], size[h] = (p * v[:, g]).sum(0), (p * v[:, g]).abs().sum(0)
    return out, size


def _bound(c, want, size, operand=2.0 ** -16):
    dim = c["q"].shape[3]
    n = int(c["lengths"].max()) + c["q"].shape[1]
    kn = c["k_pool"].float()
    kn = kn[torch.isfinite(kn).all(3)].norm(dim=1).max().double()
    score = dim ** -0.5 * c["q"].double().norm(dim=3).max() * kn * (dim + 8) * 2.0 ** -24 + \
        2.0 ** -22
    return want.abs() * 2.0 ** -8 + size * (2 * score + operand + (n + 8) * 2.0 ** -24) + 1e-30


def _check(c, dev, at, err=None, **kw):
    """*at*: pairs of a row and a node."""
    out = tree.attention(**{k: v.to(dev) for k, v in c.items()}, err=err, **kw).cpu().double()
    operand = 2.0 ** (-8 if kw.get("rounded") else -16)
    for b, t in at:
        want, size = _node(c, b, t)
        got, far = out[b, t], ~torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, t)
        there = far & ~torch.isnan(want)
        assert torch.equal(got[there], want[there]), (b, t)
        off = (got - want).abs()[~far]
        assert (off <= _bound(c, want, size, operand)[~far]).all(), (b, t, off.max())


def _some(rows, nodes):
    return sorted({(b, t) for b in (0, rows // 2, rows - 1) for t in
                   (0, nodes // 3, nodes // 2, nodes - 2, nodes - 1) if t >= 0})


@pytest.mark.parametrize("shape,form", MANY)
def test_every_form_holds_probabilities_to_16_bits(gpu_device, shape, form):
    c = _shape(shape)
    assert _form(c)[0] == 0
    _check(c, gpu_device, _some(*shape[:2]))


@pytest.mark.parametrize("shape,form", FORMS)
def test_probabilities_rounded_to_8_bits_where_asked(gpu_device, shape, form):
    """By many columns alone: by few there is nothing to gain and nothing changes."""
    c = _shape(shape)
    _check(c, gpu_device, _some(*shape[:2]), rounded=True)
    d = {k: v.to(gpu_device) for k, v in c.items()}
    assert torch.equal(tree.attention(**d, rounded=True), tree.attention(**d)) == (form[0] > 0)


@pytest.mark.parametrize("shape,form", FORMS)
def test_cached_values_that_are_not_finite(gpu_device, shape, form):
    """In the first, a middle and the last cached positions, in dims and heads of their own, both
    infinities in one dim, and beside drafted ones."""
    c = _shape(shape)
    rows, nodes, heads, kv_heads, dim, _ = shape
    for b in (0, rows - 1):
        L = int(c["lengths"][b])
        for pos, h, d, x in ((0, 0, 3, math.inf), (L // 2, 0, 8, -math.inf),
                             (L - 1, kv_heads - 1, dim - 1, math.nan), (L - 1, 0, 20, math.inf),
                             (L // 3, kv_heads - 1, 33, math.inf),
                             (L // 2, kv_heads - 1, 33, -math.inf),
                             (L // 4, 0, 50, -1e30), (L // 2, 0, 51, math.inf),
                             (L + nodes - 1, 0, 51, -math.inf), (L + nodes - 1, 0, 52, -math.inf)):
            page, off = _place(c, b, pos)
            c["v_pool"][page, h, off, d] = x
    _check(c, gpu_device, _some(rows, nodes))


@pytest.mark.parametrize("nodes", [3, 80])
def test_infinite_values_of_little_weight(gpu_device, nodes):
    """The weight of an infinite value is far below an f32's smallest number, in its own wave, split
    or tile and in others: it is above zero all the same."""
    for at in (0, 700, 1399):
        c = _case(at + nodes, 1, nodes, 2, 1, 128, [1400])
        c["q"] *= 8
        page, off = _place(c, 0, at)
        c["k_pool"][page, :, off] = c["q"][0, 0, 0] * 0.5
        for pos, d in ((3, 1), (690, 2), (710, 3), (1390, 4)):
            page, off = _place(c, 0, pos)
            c["v_pool"][page, 0, off, d] = math.inf if d % 2 else -math.inf
        _check(c, gpu_device, [(0, 0), (0, nodes - 1)])


@pytest.mark.parametrize("shape,form", FORMS)
def test_positions_in_pages_out_of_range_take_no_part(gpu_device, shape, form):
    """No page, one past the pool and a negative one, in the first, middle and last places of rows,
    drafted positions among them; the pool's first page, which no row has, holds NaN."""
    c = _shape(shape)
    rows, nodes = shape[:2]
    spare = set(range(c["k_pool"].shape[0])) - set(c["table"].flatten().tolist())
    if 0 not in spare:
        page = spare.pop()
        c["k_pool"][page], c["v_pool"][page] = c["k_pool"][0], c["v_pool"][0]
        c["table"][c["table"] == 0] = page
    c["k_pool"][0] = c["v_pool"][0] = math.nan
    pages = c["k_pool"].shape[0]
    bad = [-1, pages, -7, 2 ** 31 - 1]
    for b, width in ((0, 333 + nodes), (rows - 1, int(c["lengths"][rows - 1]) + nodes)):
        last = (width - 1) // 16
        for i, place in enumerate({0, 1, 2, last // 2, last - 1, last}):
            if 0 <= place <= last and (i + b) % 3 != 2:
                c["table"][b, place] = bad[(i + b) % 4]
    err = torch.zeros(1, dtype=I32, device=gpu_device)
    _check(c, gpu_device, _some(rows, nodes), err)
    assert err.item() == _lib.ERR_PAGE_RANGE
    c["table"][0] = -1
    d = {k: v.to(gpu_device) for k, v in c.items()}
    assert not tree.attention(**d)[0].any()


def _long(rows, nodes, heads, kv_heads, dim, lengths, far):
    """Rows of *lengths*, those of *far* by shuffled pages; the others have pages of their own up
    to theirs."""
    g = _gen(sum(lengths))
    need = [-(-(n + nodes) // 16) for n in lengths]
    pages = sum(need) + 1
    order, width = torch.randperm(pages, generator=g).to(I32), max(need)
    table, at = torch.full((rows, width), -1, dtype=I32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    parents = torch.clamp(torch.arange(nodes) - 1 - torch.arange(nodes) % 3, min=-1)
    masks = R.words(R.ancestors(parents.view(1, nodes))[0], nodes).repeat(rows, 1, 1)
    pools = [torch.randn(pages, kv_heads, 16, dim, generator=g, dtype=torch.float32).to(BF)
             for _ in range(2)]
    return {"q": torch.randn(rows, nodes, heads, dim, generator=g).to(BF), "k_pool": pools[0],
            "v_pool": pools[1], "table": table, "lengths": torch.tensor(lengths, dtype=I32),
            "masks": masks}


@pytest.mark.parametrize("rows,heads,dim,long", [
    (64, 16, 64, (4095, 4097, 8190)), (64, 16, 128, (4090, 4100, 8300)),
    (40, 32, 128, (4096, 4120, 4200)), (64, 16, 256, (4100, 4099, 8200))])
def test_few_columns_past_the_pages_a_wave_holds(gpu_device, rows, heads, dim, long):
    """A wave of four holds the pages of 32 tiles of 32 positions: 4,096 of a row that is one
    split."""
    lengths = [13 + b % 40 for b in range(rows)]
    far = (0, rows // 2, rows - 1)
    for b, n in zip(far, long):
        lengths[b] = n
    c = _long(rows, 3, heads, 8, dim, lengths, far)
    form = _form(c)
    assert form[:2] == (1, 4) and form[3] == 1, form
    _check(c, gpu_device, [(b, t) for b in far for t in range(3)])
    c["table"][far[2], 257] = -1                     # behind the refill
    _check(c, gpu_device, [(far[2], t) for t in range(3)])


@pytest.mark.parametrize("rows,nodes,heads,dim,long,waves", [
    (17, 66, 16, 64, (16390, 16384, 17000), 8), (17, 65, 16, 128, (16320, 16500, 32900), 8),
    (33, 17, 32, 64, (16384, 16450, 16400), 4), (17, 40, 32, 256, (16300, 16390, 16900), 8)])
def test_many_columns_past_the_pages_a_block_holds(gpu_device, rows, nodes, heads, dim, long,
                                                   waves):
    """A block holds 1,024 pages: 16,384 positions of a row that is one split."""
    lengths = [13 + b % 40 for b in range(rows)]
    far = (0, rows // 2, rows - 1)
    for b, n in zip(far, long):
        lengths[b] = n
    c = _long(rows, nodes, heads, 8, dim, lengths, far)
    form = _form(c)
    assert form[:2] == (0, waves) and form[3] == 1, form
    _check(c, gpu_device, [(b, t) for b in far for t in (0, nodes // 2, nodes - 1)])
    c["table"][far[2], 1026] = -1                    # behind the refill
    _check(c, gpu_device, [(far[2], t) for t in (0, nodes - 1)])


@pytest.mark.parametrize("shape,form", FORMS)
def test_nodes_that_are_not_there_are_not_written(gpu_device, shape, form):
    """Rows with one node, half of theirs, whole and without: the others' outputs hold what
    they held."""
    c = _shape(shape)
    rows, nodes, heads, kv_heads, dim, _ = shape
    counts = torch.tensor([(nodes, 0, 1, nodes // 2)[(b + 3 - (rows > 1)) % 4] for b in range(rows)],
                          dtype=I32)
    d = {k: v.to(gpu_device) for k, v in c.items()}
    held = torch.full_like(d["q"], 777.0)
    counts_d = counts.to(gpu_device)
    need = lib().tfd_tree_attn_work_bytes(rows, nodes, heads, kv_heads, dim, c["table"].shape[1])
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu_device)
    whole = tree.attention(**d, counts=counts_d)
    a = _lib.TfdTreeAttnArgs(
        ptr(d["q"]), *d["q"].stride()[:3], ptr(d["k_pool"]), ptr(d["v_pool"]), ptr(d["table"]),
        ptr(d["lengths"]), ptr(counts_d), ptr(d["masks"]), rows, nodes, heads, kv_heads, dim,
        c["table"].shape[1], c["k_pool"].shape[0], dim ** -0.5, ptr(held), 0, ptr(work), need, 0)
    lib().tfd_tree_attn(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    there = (torch.arange(nodes) < counts.unsqueeze(1)).to(gpu_device)
    assert (held[~there] == 777.0).all() and (~there).any()
    assert torch.equal(held[there], whole[there])
    for b in {0, rows // 2, rows - 1}:
        for t in {0, int(counts[b]) - 1}:
            if 0 <= t < counts[b]:                   # (a node's ancestors lie before it)
                want, size = _node(c, b, t)
                assert ((held[b, t].cpu().double() - want).abs() <= _bound(c, want, size)).all()
