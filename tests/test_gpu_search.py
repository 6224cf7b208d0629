"""Beam search and checked drafts on the batched engine: every step's choice against the
definition given the step's own logits, every row's cached positions against what was written
for them, and the tokens against greedy decoding."""
import pytest
import torch

from tests import _search_ref as R
from tests.test_gpu_engine import SMALL, _prompt
from tilefoundry_amd.qwen3 import QWEN3_1_7B, synthetic_weights
from tilefoundry_amd.qwen3.batch_engine import BatchEngine
from tilefoundry_amd.qwen3.search import NgramDraft

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights():
    """A varied greedy stream whose picks lie well apart (2.7% of the largest logit)."""
    return synthetic_weights(SMALL, seed=3, sigma=0.05, norms="ones")


def _engine(w, dev, batch, **kw):
    return BatchEngine(SMALL, w, batch=batch, device=dev,
                       **{"max_new": 40, "prompt_room": 40, **kw})


def _row(e, r, n):
    """Row r's cached keys and values [2, n, layers, heads, dim] at positions 0 .. n - 1."""
    at = torch.arange(n, device=e.device)
    page, off = e.page_table[r, at // 16].long(), at % 16
    return torch.stack((e.kpool[:, page, :, off], e.vpool[:, page, :, off])).cpu()


@pytest.mark.parametrize("groups,beams,eos,penalty", [(1, 4, None, 0.0), (3, 2, 17, 0.7),
                                                      (2, 5, 17, 0.0)])
def test_beam_steps(gpu_device, weights, groups, beams, eos, penalty):
    """Step by step: the choice from the step's logits, histories, and the cache behind
    forks and copies."""
    e = _engine(weights, gpu_device, groups * beams, graph=False)
    prompts = [_prompt(n, SMALL.vocab_size, seed=n) for n in (9, 30, 1)[:groups]]
    e.beam_search(prompts, 1, beams=beams, eos=eos, length_penalty=penalty)
    search = e._beam_searches[(beams, eos, penalty)]
    table = e.page_table.clone()
    search._begin(prompts)
    n = [len(p) - 1 for p in prompts for _ in range(beams)]
    kept = [_row(e, r, n[r]) for r in range(e.B)]
    history = [[] for _ in range(e.B)]
    for _ in range(36):
        before = [t.cpu().clone() for t in (search.scores, search.lengths, search.done)]
        # the step appends through the table as take() leaves it: read before the fork
        search.cache.take(e.pos, 1)
        shadow = e.page_table.clone()
        search._step()
        parents, tokens, scores, lengths, done = R.beam(e.logits.cpu(), *before, eos=eos,
                                                        penalty=penalty)
        assert torch.equal(search.lengths.cpu(), lengths)
        assert torch.equal(search.done.cpu(), done)
        s = search.scores.cpu().double()
        assert ((s == scores) | ((s - scores).abs() <= scores.abs() * 2.0 ** -23 + 2e-6)).all()
        new = []
        now = e.page_table.clone()
        e.page_table.copy_(shadow)
        for r in range(e.B):
            new.append(torch.cat((kept[r], _row(e, r, n[r] + 1)[:, n[r]:]), 1))
        e.page_table.copy_(now)
        kept = [new[p] for p in parents.view(-1).tolist()]
        history = [history[p] + [t] for p, t in zip(parents.view(-1).tolist(),
                                                    tokens.view(-1).tolist())]
        n = [v + 1 for v in n]
        assert e.pos.tolist() == n
        for r in range(e.B):
            assert torch.equal(_row(e, r, n[r]), kept[r]), r
    for r in range(e.B):
        start = len(prompts[r // beams]) - 1
        assert e.sam[r, start:start + 36].tolist() == history[r]
    # forked rows share pages, and none is lost
    refs = torch.zeros_like(search.cache.refs)
    used = e.page_table.flatten().long()
    refs.scatter_add_(0, used[used >= 0], torch.ones_like(used[used >= 0], dtype=refs.dtype))
    assert torch.equal(refs, search.cache.refs)
    search.cache.check_errors()
    e.page_table.copy_(table)


def test_one_beam_is_greedy_and_graphs_change_nothing(gpu_device, weights):
    prompts = [_prompt(n, SMALL.vocab_size, seed=20 + n) for n in (12, 7)]
    e = _engine(weights, gpu_device, 2)
    greedy = e.generate(prompts, 24, prefill=True).tokens
    one = e.beam_search(prompts, 24, beams=1)
    assert [b[0] for b in one.tokens] == greedy
    two = e.beam_search(prompts[:1], 24, beams=2)
    assert e.generate(prompts, 24, prefill=True).tokens == greedy     # the table is put back
    again = e.beam_search(prompts[:1], 24, beams=2)
    plain = _engine(weights, gpu_device, 2, graph=False).beam_search(prompts[:1], 24, beams=2)
    for r in (again, plain):
        assert r.tokens == two.tokens and r.scores == two.scores
    assert two.scores[0][0] >= two.scores[0][1]
    assert len(two.tokens[0][0]) == 24


def test_beams_end_at_eos(gpu_device, weights):
    prompt = _prompt(10, SMALL.vocab_size, seed=5)
    e = _engine(weights, gpu_device, 4)
    free = e.beam_search([prompt], 20, beams=4)
    eos = free.tokens[0][0][6]
    got = e.beam_search([prompt], 20, beams=4, eos=eos, length_penalty=1.0)
    ended = [t for t, f in zip(got.tokens[0], got.finished[0]) if f]
    assert ended and all(t[-1] == eos and eos not in t[:-1] for t in ended)


class _Known:
    """A draft that knows the continuation, behind a wrong branch of its own if asked."""

    def __init__(self, prompts, truth, wrong):
        self.full = [list(p) + list(t) for p, t in zip(prompts, truth)]
        self.wrong = wrong

    def __call__(self, history, nodes):
        full = next(f for f in self.full if f[:len(history)] == list(history))
        right = full[len(history):]
        tokens, parents = [history[-1]], [-1]
        if self.wrong and len(tokens) < nodes and right:
            tokens.append((right[0] + 1) % SMALL.vocab_size)
            parents.append(0)
        node = 0
        for t in right[:nodes - len(tokens)]:
            tokens.append(t)
            parents.append(node)
            node = len(tokens) - 1
        return tokens, parents


@pytest.mark.parametrize("nodes", [1, 5, 16, 40])
def test_speculation_gives_the_greedy_tokens(gpu_device, weights, nodes):
    prompts = [_prompt(n, SMALL.vocab_size, seed=40 + n) for n in (16, 3, 33)]
    e = _engine(weights, gpu_device, 3)
    want = e.generate(prompts, 30, prefill=True).tokens
    for draft in (NgramDraft(), NgramDraft(2, 3), _Known(prompts, want, False),
                  _Known(prompts, want, True), lambda h, n: ([h[-1], 5, 5][:n], [-1, 0, 1][:n])):
        got = e.speculate(prompts, 30, nodes=nodes, draft=draft)
        assert got.tokens == want
    known = e.speculate(prompts, 30, nodes=nodes, draft=_Known(prompts, want, False))
    assert known.passes == -(-30 // nodes)
    assert e.generate(prompts, 30, prefill=True).tokens == want


def test_speculation_without_graphs(gpu_device, weights):
    """The captured pass and its launches one by one give the same, again and again."""
    prompts = [_prompt(n, SMALL.vocab_size, seed=80 + n) for n in (21, 6)]
    plain = _engine(weights, gpu_device, 2, graph=False)
    e = _engine(weights, gpu_device, 2)
    for nodes in (6, 9, 6):
        want = plain.speculate(prompts, 30, nodes=nodes)
        for _ in range(3):
            got = e.speculate(prompts, 30, nodes=nodes)
            assert got.tokens == want.tokens and got.passes == want.passes
            e.generate(prompts, 5, prefill=True)     # eager work and the step's graph between


def test_speculation_with_room_for_many_nodes(gpu_device, weights):
    prompts = [_prompt(n, SMALL.vocab_size, seed=40 + n) for n in (16, 3, 33)]
    e = _engine(weights, gpu_device, 3)
    want = e.generate(prompts, 30, prefill=True).tokens
    assert e.speculate(prompts, 30, nodes=200, draft=_Known(prompts, want, True)).tokens == want


def test_prompts_of_one_token_and_one_new(gpu_device, weights):
    e = _engine(weights, gpu_device, 2)
    for prompts in ([[5], [9]], [[5], [9, 3]]):
        want = e.generate(prompts, 6).tokens
        assert e.speculate(prompts, 6, nodes=4).tokens == want
        assert [b[0] for b in e.beam_search(prompts, 6, beams=1).tokens] == want
        assert [len(t) for t in e.speculate(prompts, 1).tokens] == [1, 1]
    two = e.beam_search([[5]], 1, beams=2)
    assert two.tokens[0][0] == e.generate([[5], [9]], 1).tokens[0] and len(two.tokens[0][1]) == 1


def test_searches_up_to_the_last_position(gpu_device, weights):
    """Prompt and new tokens fill the engine's steps: the last node's slot is the last one."""
    e = _engine(weights, gpu_device, 2, max_new=14, prompt_room=20)
    prompts = [_prompt(20, SMALL.vocab_size, seed=n) for n in (60, 61)]
    run = e.generate(prompts, 14, prefill=True, record_logits=True)
    for draft in (NgramDraft(), _Known2(prompts, run.tokens)):
        got = e.speculate(prompts, 14, nodes=16, draft=draft)
        for b in range(2):
            _same_to_a_near_tie(run.tokens[b], run.logits[b], got.tokens[b])
    got = e.beam_search(prompts, 14, beams=1)
    for b in range(2):
        _same_to_a_near_tie(run.tokens[b], run.logits[b], got.tokens[b][0])


def _same_to_a_near_tie(want, logits, got):
    assert len(want) == len(got)
    differ = [i for i, (a, b) in enumerate(zip(want, got)) if a != b]
    if differ:
        at = logits[differ[0]]
        assert 0 <= float(at[want[differ[0]]] - at[got[differ[0]]]) <= 2e-2 * float(at.abs().max())


def test_speculation_of_text_that_repeats(gpu_device, weights):
    """Fewer passes where the n-gram draft finds something, and the greedy tokens up to the first
    near-tie.

    This stream has an exact one: behind 24 tokens the bf16 logits of 2471 and 3053 are both
    3.0156, so the pick rests on the order of two sums that both rounded to it, and a step and a
    pass sum in different orders.  At the first difference the two tokens' logits may therefore
    differ by what two orders can move them: 2% of the largest, the margin that the other streams
    of these tests keep."""
    prompt = _prompt(6, SMALL.vocab_size, seed=1) * 5
    e = _engine(weights, gpu_device, 1, max_new=60)
    run = e.generate([prompt], 60, prefill=True, record_logits=True)
    got = e.speculate([prompt], 60, nodes=8)
    assert got.passes <= 60 and len(got.tokens[0]) == 60
    _same_to_a_near_tie(run.tokens[0], run.logits[0], got.tokens[0])


def test_speculation_at_the_qwen3_layer_shape(gpu_device):
    cfg = QWEN3_1_7B.with_(num_hidden_layers=2)
    w = synthetic_weights(cfg, seed=3, sigma=0.05, norms="ones")
    e = BatchEngine(cfg, w, batch=2, device=gpu_device, max_new=12, prompt_room=40)
    prompts = [_prompt(n, cfg.vocab_size, seed=n) for n in (33, 8)]
    run = e.generate(prompts, 12, prefill=True, record_logits=True)
    got = e.speculate(prompts, 12, nodes=6, draft=_Known2(prompts, run.tokens))
    for b in range(2):
        _same_to_a_near_tie(run.tokens[b], run.logits[b], got.tokens[b])


class _Known2(_Known):
    def __init__(self, prompts, truth):
        super().__init__(prompts, truth, False)

    def __call__(self, history, nodes):              # (nothing to know behind another pick)
        if not any(f[:len(history)] == list(history) for f in self.full):
            return [history[-1]], [-1]
        return super().__call__(history, nodes)


def test_searches_refuse(gpu_device, weights):
    from tilefoundry_amd.sampling import Sampling

    e = _engine(weights, gpu_device, 4)
    p = [1, 2, 3]
    for call, match in (
            (lambda: e.beam_search([p], 8, beams=3), "divide"),
            (lambda: e.beam_search([p, p], 8, beams=4), "1 non-empty"),
            (lambda: e.beam_search([[]], 8, beams=4), "non-empty"),
            (lambda: e.beam_search([p], 0, beams=4), "max_new"),
            (lambda: e.beam_search([p], 1000, beams=4), "exceeds"),
            (lambda: e.beam_search([[SMALL.vocab_size]], 8, beams=4), "ids"),
            (lambda: e.beam_search([p], 8, beams=4, eos=SMALL.vocab_size), "eos"),
            (lambda: e.speculate([p], 8), "4 non-empty"),
            (lambda: e.speculate([p] * 4, 8, nodes=0), "nodes"),
            (lambda: e.speculate([p] * 4, 8, nodes=257), "nodes"),
            (lambda: e.speculate([p] * 4, 8, draft=lambda h, n: ([1, 2], [-1, 0])), "draft"),
            (lambda: e.speculate([p] * 4, 8, draft=lambda h, n: ([h[-1], -4], [-1, 0])), "ids"),
            (lambda: e.speculate([p] * 4, 8, draft=lambda h, n: ([h[-1]], [-1, 0])), "parents"),
            (lambda: e.speculate([p] * 4, 8, draft=lambda h, n: ([h[-1], 3, 4], [-1, 2, 0])),
             "before it"),
            (lambda: e.speculate([p] * 4, 8, draft=lambda h, n: ([h[-1], 3], [0, 0])),
             "before it")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(ValueError, match="pass"):
        _engine(weights, gpu_device, 17).speculate([p] * 17, 4, nodes=256)
    with pytest.raises(ValueError, match="greedy"):
        _engine(weights, gpu_device, 1, sampling=Sampling(top_k=4)).speculate([p], 4)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("groups,beams", [(1, 4), (2, 3)])
def test_beam_steps_take_their_own_pages(gpu_device, weights, monkeypatch, groups, beams, graph):
    """Nothing but the step takes pages: its table is looked at between its take and its fork (one
    by one), and every row's cache behind the fork is its parent's with what was written for that,
    also where the captured step is replayed."""
    e = _engine(weights, gpu_device, groups * beams, graph=graph)
    prompts = [_prompt(n, SMALL.vocab_size, seed=n) for n in (9, 30)[:groups]]
    e.beam_search(prompts, 1, beams=beams)
    search = e._beam_searches[(beams, None, 0.0)]
    assert (search.graph is not None) == graph
    table, taken = e.page_table.clone(), torch.zeros_like(e.page_table)
    chosen = torch.zeros(e.B, dtype=torch.int32, device=e.device)
    forward, fork = e._forward, search.cache.fork

    def look(s):
        taken.copy_(e.page_table)
        forward(s)

    def follow(parents, lengths):
        chosen.copy_(parents)
        return fork(parents, lengths)

    monkeypatch.setattr(e, "_forward", look)
    monkeypatch.setattr(search.cache, "fork", follow)
    if graph:
        search._capture()                            # (with what looks at it in it)
    search._begin(prompts)
    n = [len(p) - 1 for p in prompts for _ in range(beams)]
    kept, shared = [_row(e, r, n[r]) for r in range(e.B)], 0
    for _ in range(36):
        shared += int((search.cache.refs > 1).sum())
        if graph:
            search.graph.replay()
        else:
            search._step()
        after, parents = e.page_table.clone(), chosen.tolist()
        e.page_table.copy_(taken)
        rows = [_row(e, r, n[r] + 1) for r in range(e.B)]
        last = [int(taken[r, n[r] // 16]) for r in range(e.B)]
        assert len(set(last)) == e.B                 # a page of one's own to write
        e.page_table.copy_(after)
        for r in range(e.B):
            assert torch.equal(rows[r][:, :n[r]], kept[r]), r
        n = [v + 1 for v in n]
        assert e.pos.tolist() == n
        kept = [rows[p] for p in parents]
        for r in range(e.B):
            assert torch.equal(_row(e, r, n[r]), kept[r]), r
    assert shared > 0
    search.cache.check_errors()
    e.page_table.copy_(table)


def test_a_refused_search_costs_no_other(gpu_device, weights):
    """An engine's searches stay where another one is refused."""
    e = _engine(weights, gpu_device, 4)
    rules = [(1, None), (2, None), (4, None), (4, 5)]
    for beams, eos in rules:
        e.beam_search([[1, 2]] * (4 // beams), 2, beams=beams, eos=eos)
    known = dict(e._beam_searches)
    for kw in ({"beams": 3}, {"beams": 0}, {"beams": 4, "eos": SMALL.vocab_size},
               {"beams": 2, "length_penalty": -1.0}):
        with pytest.raises(ValueError):
            e.beam_search([[1, 2]], 2, **kw)
    assert e._beam_searches == known
    e.speculate([[1, 2]] * 4, 2, nodes=3)
    one = e._speculations[3]
    with pytest.raises(ValueError):
        e.speculate([[1, 2]] * 4, 2, nodes=0)
    assert e._speculations == {3: one}
