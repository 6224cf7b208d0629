"""Beams against every candidate sorted in 64 bits: parents, tokens, lengths and done equal;
scores within one f32 rounding (2^-24) of the value and of the 64-bit sum's noise, whose terms
are f32 exponentials (2^-22 each, relative, of a sum: as much in its logarithm)."""
import math

import pytest
import torch

from tests import _search_ref as R
from tilefoundry_amd import _lib
from tilefoundry_amd.beam import Beam, States

pytestmark = pytest.mark.gpu

F32, BF, F16, I32 = torch.float32, torch.bfloat16, torch.float16, torch.int32


def _check(dev, rule, logits, scores, lengths=None, done=None):
    d = [None if t is None else t.to(dev) for t in (logits, scores, lengths, done)]
    got = rule(*d)
    want = R.beam(logits, scores, lengths, done, eos=rule.eos, penalty=rule.length_penalty)
    for name, a, b in zip(("parents", "tokens", "lengths", "done"),
                          (got.parents, got.tokens, got.lengths, got.done),
                          (want[0], want[1], want[3], want[4])):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name
    s, w = got.scores.cpu().double(), want[2]
    assert ((s == w) | ((s - w).abs() <= w.abs() * 2.0 ** -24 + 2.0 ** -22)).all()
    return got


def _draw(seed, groups, beams, vocab, dtype=F32):
    """Logits whose candidates lie well apart: the order of two rows' sums does not hang on
    a rounding."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(groups * beams, vocab, generator=g) * 2
    return x.to(dtype), -10 + torch.randn(groups, beams, generator=g), g


@pytest.mark.parametrize("groups,beams,vocab,dtype", [
    (1, 1, 1, F32), (1, 3, 2, F32), (2, 4, 5, BF), (1, 4, 1000, F32), (3, 5, 1023, F16),
    (2, 8, 4099, F32), (1, 64, 700, F32), (1, 33, 30000, BF), (5, 2, 151936, F32),
    (1, 4, 262144, F16), (40, 16, 3001, F32)])
def test_beam_matches_definition(gpu_device, groups, beams, vocab, dtype):
    x, s, g = _draw(vocab + beams, groups, beams, vocab, dtype)
    _check(gpu_device, Beam(beams), x, s)
    lengths = torch.randint(0, 50, s.shape, generator=g, dtype=I32)
    done = torch.rand(s.shape, generator=g) < 0.3
    for penalty in (0.0, 0.7, 1.0):
        _check(gpu_device, Beam(beams, eos=vocab // 2, length_penalty=penalty), x, s, lengths,
               done)


def test_beam_first_step_takes_one_row(gpu_device):
    """A search starts with one beam a group: the others' scores are minus infinity."""
    x, s, _ = _draw(1, 3, 6, 500)
    s[:, 1:] = -math.inf
    got = _check(gpu_device, Beam(6), x, s)
    assert (got.parents.cpu() == torch.arange(3).unsqueeze(1) * 6).all()


def test_beam_ties_go_to_the_lower_row_then_token(gpu_device):
    """Equal logits all over (thousands of candidates of one rank), and equal ones in a row."""
    for groups, beams, vocab in ((1, 4, 40), (2, 16, 20000), (1, 64, 9000)):
        x = torch.zeros(groups * beams, vocab)
        got = _check(gpu_device, Beam(beams, eos=1), x, torch.zeros(groups, beams))
        assert (got.tokens.cpu()[:, :vocab] == torch.arange(beams)[:vocab]).all()
    g = torch.Generator().manual_seed(3)
    x = torch.randint(0, 4, (8, 5000), generator=g).float()
    _check(gpu_device, Beam(8), x, torch.arange(8.0).view(1, 8) * -0.37)
    x = torch.zeros(4, 300)
    x[:, ::2] = -0.0
    _check(gpu_device, Beam(4), x, torch.zeros(1, 4))


def test_beam_masks_infinities_and_nan(gpu_device):
    """Rows with no candidate, one, fewer than beams; NaN; the types' lowest value; +inf."""
    K, V = 8, 3000
    x, s, _ = _draw(4, 2, K, V)
    x[0] = -math.inf
    x[1] = math.nan
    x[2] = -math.inf
    x[2, 1717] = 3.0
    x[3, ::3] = math.nan
    x[4] = torch.finfo(F32).min
    x[4, 7] = 0.0
    x[5, 11] = x[5, 2900] = math.inf
    s[0, 6] = math.nan
    s[0, 7] = math.inf
    x[8:] = -math.inf                                # a group with three candidates in all
    x[9, 5] = x[12, 6] = x[12, 4] = 1.0
    lengths = torch.arange(16, dtype=I32).view(2, 8)
    done = torch.zeros(2, 8, dtype=torch.bool)
    got = _check(gpu_device, Beam(K, eos=4), x, s, lengths, done)
    assert (got.tokens[1, 3:] == -1).all() and (got.scores[1, 3:] == -math.inf).all()
    done[1, 2] = True
    _check(gpu_device, Beam(K, eos=4, length_penalty=0.5), x, s, lengths, done)
    _check(gpu_device, Beam(K), x, s, lengths, done)
    done[:] = True
    _check(gpu_device, Beam(K, eos=4), x, s, lengths, done)


@pytest.mark.parametrize("groups,beams,vocab,dtype", [
    (1, 64, 151936, BF), (2, 64, 40000, F32), (4, 32, 100352, F32), (3, 16, 100352, BF),
    (2, 24, 20000, F16), (2, 25, 20000, F16), (1, 64, 40001, F32), (1, 64, 40001, BF)])
def test_beam_rows_that_offer_much(gpu_device, groups, beams, vocab, dtype):
    """Many beams; one row far ahead, whose lists hold more candidates than there are lists; all
    rows alike but for their logits."""
    x, s, _ = _draw(vocab - beams, groups, beams, vocab, dtype)
    _check(gpu_device, Beam(beams), x, s)
    s[:, beams // 2] += 30
    _check(gpu_device, Beam(beams), x, s)
    s[:] = -1.5
    _check(gpu_device, Beam(beams), x, s)


@pytest.mark.parametrize("beams", [4, 16, 64])
def test_beam_thousands_of_equal_logits(gpu_device, beams):
    x = torch.zeros(beams, 30000)
    s = -torch.arange(float(beams)).view(1, beams)
    _check(gpu_device, Beam(beams), x, s)            # a row's lowest tokens first
    x[:] = -3e38                                     # masked but for three tokens a row
    x[:, [17, 9000, 29999]] = torch.tensor([1.0, 2.0, 0.5])
    s = s * 0.25
    # Rows r and r + 2 differ by the half that logits 1.0 and 0.5 do: their candidates are equal
    # in exact arithmetic (-r / 4 + 0.5 = -(r + 2) / 4 + 1.0), and which of two such is
    # larger in 64 bits hangs on where the sum with lse was rounded (2^-53).  Their order is
    # left open; values, the candidates' own values and that each comes once are not.
    got = Beam(beams)(x.to(gpu_device), s.to(gpu_device))
    want = R.beam(x, s, None, None)[2]
    assert ((got.scores.cpu().double() - want).abs() <= want.abs() * 2.0 ** -24 + 2.0 ** -22).all()
    p, t = got.parents.cpu()[0].long(), got.tokens.cpu()[0].long()
    own = s[0, p].double() + torch.log_softmax(x.double(), 1)[p, t]
    assert ((own - want[0]).abs() <= 2.0 ** -40).all()
    assert len(set(zip(p.tolist(), t.tolist()))) == beams


@pytest.mark.parametrize("scale", [1e4, 9e5, 3e6, 1e30])
def test_beam_large_logits(gpu_device, scale):
    """A reference whose product with log2 e is rounded by as much as the differences are."""
    x, s, _ = _draw(8, 2, 4, 9001)
    _check(gpu_device, Beam(4), x + scale, s)
    _check(gpu_device, Beam(4), x - scale, s)


def test_beam_adversarial_places(gpu_device):
    """The best logits side by side, all in one thread's or one chunk's values."""
    for at in (0, 4, 1021, 9000):
        x, s, _ = _draw(at, 1, 32, 12000)
        x[:, at:at + 200] += 40
        _check(gpu_device, Beam(32), x, s)
    x = torch.arange(12000.0).repeat(16, 1) * 1e-3   # rising and falling rows
    x[8:] = x[8:].flip(1)
    _check(gpu_device, Beam(16), x, torch.arange(16.0).view(1, 16) * -0.0501)


def test_beam_strides_streams_and_graphs(gpu_device):
    x, s, g = _draw(8, 2, 4, 1500)
    rule = Beam(4, eos=3)
    want = rule(x.to(gpu_device), s.to(gpu_device))
    wide = torch.zeros(8, 1511, device=gpu_device)
    wide[:, 5:1505] = x.to(gpu_device)
    turned = x.to(gpu_device).t().contiguous().t()
    for y in (wide[:, 5:1505], turned):
        for a, b in zip(rule(y, s.to(gpu_device)), want):
            assert torch.equal(a, b)
    xd, sd = x.to(gpu_device), s.to(gpu_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rule(xd, sd)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rule(xd, sd)
    for k in range(3):
        xd.copy_(torch.randn(8, 1500, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, rule(xd, sd)):
            assert torch.equal(a, b)


def test_beam_empty(gpu_device):
    got = Beam(4)(torch.zeros(0, 9, device=gpu_device), torch.zeros(0, 4, device=gpu_device))
    assert got.parents.shape == (0, 4)


@pytest.mark.parametrize("groups,beams,shapes", [
    (1, 1, [(4,)]), (1, 4, [(2176,), (3, 5)]), (3, 5, [(33,), (1,)]), (2, 8, [(4, 4, 16)]),
    (2, 16, [(1000,), (7,)]), (1, 32, [(513,)]), (2, 64, [(129,), (4096,)])])
def test_reorder(gpu_device, groups, beams, shapes):
    rows = groups * beams
    g = torch.Generator().manual_seed(rows)
    kinds = [F32, BF, torch.uint8, I32, torch.float64]
    own = [torch.randint(0, 250, (rows, *shape), generator=g).to(t) for shape in shapes
           for t in kinds]
    d = [t.to(gpu_device) for t in own]
    states = States(d, beams)
    for k in range(4):
        parents = torch.randint(0, beams, (groups, beams), generator=g)
        if k == 1:
            parents[:] = torch.arange(beams).flip(0)         # pairs change places
        if k == 2:
            parents[:] = torch.arange(beams)
        parents = (parents + beams * torch.arange(groups).unsqueeze(1)).to(I32)
        states.reorder(parents.to(gpu_device) if k % 2 else parents.view(-1).to(gpu_device))
        own = [t[parents.view(-1).long()] for t in own]
        for a, b in zip(d, own):
            assert torch.equal(a.cpu(), b)
    states.check_errors()


def test_reorder_leaves_rows_of_bad_parents(gpu_device):
    x = torch.arange(12.0, device=gpu_device).view(4, 3)
    states = States([x], beams=2)
    states.reorder(torch.tensor([1, 2, -1, 2], dtype=I32, device=gpu_device))
    assert x.cpu()[:, 0].tolist() == [3.0, 3.0, 6.0, 6.0]
    with pytest.raises(RuntimeError, match="outside"):
        states.check_errors()
    states.check_errors()


def test_reorder_unaligned_and_captured(gpu_device):
    base = torch.arange(3 * 1001 + 1, device=gpu_device, dtype=torch.uint8)
    x = base[1:].view(3, 1001)
    h = torch.arange(3 * 77 + 1, device=gpu_device, dtype=F32).to(BF)[1:].view(3, 77)
    own = [x.clone(), h.clone()]
    states = States([x, h, torch.zeros(3, 0, device=gpu_device)])
    parents = torch.tensor([1, 2, 0], dtype=I32, device=gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        states.reorder(parents)
    for order in ([1, 2, 0], [0, 0, 0], [2, 1, 0]):
        parents.copy_(torch.tensor(order, dtype=I32))
        graph.replay()
        torch.cuda.synchronize()
        own = [t[parents.long()] for t in own]
        assert torch.equal(x, own[0]) and torch.equal(h, own[1])


def test_reorder_rows_past_4_gib(gpu_device):
    n = (1 << 32) // 4 + 1028
    x = torch.zeros(2, n, device=gpu_device)
    x[0, -3:], x[1, -3:] = 1.0, 2.0
    x[1, 5] = 7.0
    States([x]).reorder(torch.tensor([1, 0], dtype=I32, device=gpu_device))
    assert x[0, -3:].tolist() == [2.0] * 3 and x[1, -3:].tolist() == [1.0] * 3
    assert x[0, 5].item() == 7.0 and x[1, 5].item() == 0.0
    assert _lib.BEAM_MAX == 64


@pytest.mark.parametrize("penalty", [0.5, 1.0, 2.0])
@pytest.mark.parametrize("beams", [4, 32, 64])
def test_beam_equal_ranks_of_unlike_lengths(gpu_device, beams, penalty):
    """Finished beams whose scores over length ** penalty are the same number, exactly: the lower
    row first.  (Scores, lengths and their powers are whole numbers here.)"""
    n = 1 + torch.randperm(90, generator=torch.Generator().manual_seed(beams))[:beams]
    lengths = n * n if penalty == 0.5 else n
    scores = -3.0 * (n * n if penalty == 2.0 else n).float()
    got = _check(gpu_device, Beam(beams, eos=1, length_penalty=penalty), torch.zeros(beams, 9),
                 scores.view(1, -1), lengths.to(I32).view(1, -1),
                 torch.ones(1, beams, dtype=torch.bool))
    assert got.parents.cpu()[0].tolist() == list(range(beams))


@pytest.mark.parametrize("penalty", [0.6, 0.7, 1.1])
def test_beam_penalty_is_not_rounded(gpu_device, penalty):
    """Finished beams, of 3 and 2^20 tokens, whose order is one thing by the penalty and another
    by its nearest f32."""
    rounded = float(torch.tensor(penalty, dtype=F32))
    long = torch.tensor(-1000.0)
    short = (long.double() * (3 / 2 ** 20) ** penalty).float()
    ranks = [lambda p, s: float(s.double()) / 3 ** p, lambda p, s: float(long) / (2 ** 20) ** p]
    step = short
    for _ in range(40):                              # (f32 neighbours on both sides)
        step = torch.nextafter(step, torch.tensor(-math.inf))
    for _ in range(80):
        step = torch.nextafter(step, torch.tensor(math.inf))
        gap = [ranks[0](p, step) - ranks[1](p, step) for p in (penalty, rounded)]
        if gap[0] * gap[1] < 0 and abs(gap[0]) > 1e-12:
            break
    else:
        raise AssertionError("no such pair")
    for scores in ((step, long), (long, step)):
        _check(gpu_device, Beam(2, eos=1, length_penalty=penalty), torch.zeros(2, 9),
               torch.stack(scores).view(1, 2),
               torch.tensor([[3 if s is step else 2 ** 20 for s in scores]], dtype=I32),
               torch.ones(1, 2, dtype=torch.bool))
