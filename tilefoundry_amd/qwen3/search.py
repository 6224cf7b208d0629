"""More than one continuation of a sequence: beams, and drafted tokens checked together.

The reference decodes one continuation a sequence, token by token
(``examples/qwen3_1_7b-tilelang/fast/engine.py:239-271``).  Both searches here run on a
``BatchEngine`` and its cache:

* ``BeamSearch`` keeps the best ``beams`` continuations of each prompt.  A group's beams are
  rows of the engine's batch; after a step the rows' new tokens are chosen among all of a
  group's candidates (``beam.Beam``), token histories follow their rows (``beam.States``), and
  rows that continue one row share its pages until they write (``pages.Pages``).
* ``Speculation`` lets a draft propose a tree of tokens, takes all of them through the model in
  one pass (``TreePass``: attention by ``tree.attention``'s kernel), walks along the greedy picks
  that agree (``tree.accept``) and moves the accepted positions together (``Pages.keep``).  The
  tokens are those of greedy decoding, up to near-ties: a pass's products and the step's sum
  in other orders, and round attention's probabilities in other places.
"""
from __future__ import annotations

import ctypes
from time import perf_counter

import numpy as np
import torch

from .. import _lib, tree
from .._lib import ptr
from ..beam import Beam, States
from ..pages import Pages
from .prefill import MAX_PASS, Prefill, in_vocab, token_array

I32 = torch.int32


class BeamGenerated:
    """Each prompt's beams, the best first, and the search's timing."""

    def __init__(self, tokens, scores, finished, seconds, prefill_seconds, steps):
        self.tokens: list[list[list[int]]] = tokens
        self.scores: list[list[float]] = scores         # sums of log probabilities
        self.finished: list[list[bool]] = finished      # ended with the eos token
        self.seconds = seconds
        self.prefill_seconds = prefill_seconds
        self.steps = steps


def _checked(e, prompts, count: int, max_new: int):
    if e.sampling is not None:
        raise ValueError("a search is greedy: this engine samples")
    if len(prompts) != count or any(len(p) < 1 for p in prompts):
        raise ValueError(f"need {count} non-empty prompts, got {len(prompts)}")
    if max_new < 1:
        raise ValueError(f"max_new must be at least 1, got {max_new}")
    prompts = [token_array(p) for p in prompts]
    if not all(in_vocab(p, e.V) for p in prompts):
        raise ValueError(f"prompt ids must lie in [0, {e.V})")
    longest = max(len(p) for p in prompts)
    if longest + max_new > e.nsteps:
        raise ValueError(f"prompt {longest} + {max_new} new exceeds this engine's {e.nsteps} "
                         "steps")
    return prompts


class BeamSearch:
    """Beam search on a batch engine (a weak reference to it: the engine keeps its searches).

    While a search runs, the engine's page table holds the beams' shared pages; it is put back
    behind it, and the positions that were cached are lost."""

    def __init__(self, engine, beams: int, eos: int | None, length_penalty: float):
        self._engine = engine
        e = engine()
        self.rule = Beam(beams, eos=eos, length_penalty=length_penalty)
        if e.B % beams:
            raise ValueError(f"beams {beams} do not divide the engine's batch {e.B}")
        if eos is not None and eos >= e.V:
            raise ValueError(f"eos must lie in [0, {e.V}), got {eos}")
        self.groups, dev = e.B // beams, e.device
        shape = (self.groups, beams)
        self.cache = Pages([e.kpool, e.vpool], table=e.page_table)
        self.states = States([e.sam], beams)
        self.scores = torch.zeros(shape, dtype=torch.float32, device=dev)
        self.lengths = torch.zeros(shape, dtype=I32, device=dev)
        self.done = torch.zeros(shape, dtype=torch.bool, device=dev)
        self.zeros = torch.zeros(e.B, dtype=I32, device=dev)
        self.graph = None

    def _step(self):
        e = self._engine()
        s = e._stream()
        self.cache.take(e.pos, 1)
        e._forward(s)
        step = self.rule(e.logits, self.scores, self.lengths, self.done)
        self.states.reorder(step.parents)
        self.scores.copy_(step.scores)
        self.lengths.copy_(step.lengths)
        self.done.copy_(step.done)
        torch.clamp(step.tokens.view(-1), min=0, out=e.pick)   # (a place without a candidate: -1)
        e._finalize(s)
        e.pos.copy_(self.cache.fork(step.parents.view(-1), e.pos))

    def _capture(self):
        torch.cuda.synchronize(self._engine().device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step()
        self.graph = graph

    def _begin(self, prompts):
        """The prompts in their groups' first rows, shared by the others; one beam a group."""
        e, K = self._engine(), self.rule.beams
        e._load_prompts([p for p in prompts for _ in range(K)])
        self.cache.table.fill_(-1)
        self.cache.refs.zero_()
        n = torch.zeros(self.groups, K, dtype=I32)
        n[:, 0] = torch.tensor([len(p) - 1 for p in prompts], dtype=I32)
        n = n.view(-1).to(e.device)
        self.cache.take(self.zeros, n)
        e._prompt_pass().run_many([(p[:-1], 0, g * K) for g, p in enumerate(prompts) if len(p) > 1])
        first = torch.arange(e.B, dtype=I32, device=e.device) // K * K
        e.pos.copy_(self.cache.fork(first, n))
        e.ids.copy_(torch.tensor([int(p[-1]) for p in prompts for _ in range(K)],
                                 dtype=torch.int64))
        e._lib.tfd_embed_rows_bf16(ptr(e.w_embed), ptr(e.ids), ptr(e.hid), e.H, e.B, e.H, e.V,
                                   ptr(e.err), e._stream())
        self.scores.fill_(-torch.inf)
        self.scores[:, 0] = 0.0
        self.lengths.zero_()
        self.done.zero_()

    def run(self, prompts, max_new: int) -> BeamGenerated:
        e, K = self._engine(), self.rule.beams
        prompts = _checked(e, prompts, self.groups, max_new)
        table = e.page_table.clone()
        try:
            if self.graph is None and e.graph is not None:
                self._capture()
            torch.cuda.synchronize(e.device)
            t0 = perf_counter()
            self._begin(prompts)
            torch.cuda.synchronize(e.device)
            t1 = perf_counter()
            steps = 0
            for steps in range(1, max_new + 1):
                if self.graph is not None:
                    self.graph.replay()
                else:
                    self._step()
                if self.rule.eos is not None and steps % 16 == 0 and bool(self.done.all()):
                    break
            torch.cuda.synchronize(e.device)
            t2 = perf_counter()
            e.check_errors()
            self.cache.check_errors()
            self.states.check_errors()
            sam, lengths = e.sam.cpu(), self.lengths.cpu()
            tokens = [[sam[g * K + b, len(p) - 1:len(p) - 1 + int(lengths[g, b])].tolist()
                       for b in range(K)] for g, p in enumerate(prompts)]
            return BeamGenerated(tokens, self.scores.tolist(), self.done.tolist(), t2 - t1, t1 - t0,
                                 steps)
        finally:
            e.page_table.copy_(table)


class NgramDraft:
    """Drafts what followed the sequence's last tokens where they came before: of the longest
    run up to *longest* tokens that did, its latest *branches* continuations, as one tree."""

    def __init__(self, longest: int = 3, branches: int = 2):
        if longest < 1 or branches < 1:
            raise ValueError(f"longest and branches are at least 1, got {longest} and {branches}")
        self.longest, self.branches = longest, branches

    def __call__(self, history, nodes: int):
        """(tokens, parents) of up to *nodes* nodes behind *history* (node 0 is its last token)."""
        h = np.asarray(history, dtype=np.int64)
        tokens, parents = [int(h[-1])], [-1]
        for n in range(min(self.longest, len(h) - 1), 0, -1):
            windows = np.lib.stride_tricks.sliding_window_view(h[:-1], n)
            at = np.flatnonzero((windows == h[-n:]).all(1))[::-1][:self.branches] + n
            if not len(at):
                continue
            each = -(-(nodes - 1) // len(at))
            for start in at:
                node = 0
                for t in h[start:start + each].tolist():
                    child = next((c for c in range(node + 1, len(tokens))
                                  if parents[c] == node and tokens[c] == t), None)
                    if child is None:
                        if len(tokens) >= nodes:
                            break
                        child = len(tokens)
                        tokens.append(t)
                        parents.append(node)
                    node = child
            break
        return tokens, parents


class TreePass(Prefill):
    """All sequences' drafted nodes through every layer and the head together: a prompt pass whose
    rows are nodes, at the positions of their depths, with attention along their branches."""

    def __init__(self, engine, nodes: int):
        super().__init__(engine, packed=True)
        e = self.e
        self.nodes, B, dev = nodes, e.B, e.device
        M = B * nodes
        self._reserve(M)
        self.seq = torch.arange(B, dtype=I32, device=dev).repeat_interleave(nodes)
        self.at = torch.arange(nodes, dtype=I32, device=dev)
        self.logits = torch.zeros(M, e.V, dtype=torch.float32, device=dev)
        self.picks = torch.zeros(B, nodes, dtype=I32, device=dev)
        self.arg_work = torch.zeros(M * _lib.ARGMAX_WORK, dtype=I32, device=dev)
        need = self._lib.tfd_tree_attn_work_bytes(B, nodes, self.HQ, self.HKV, self.D,
                                                  self.max_pages)
        self.attn_work = torch.zeros(max(need, 16), dtype=torch.uint8, device=dev)

    def _node_layer(self, i, M, pos, slot, lengths, counts, masks, s):
        """``_layer`` (model.py:236-266) for the nodes; the last layer goes on to the head."""
        L, w, e = self._lib, self.layers[i], self.e
        H, I, table = self.H, self.I, ptr(e.page_table)
        sl = self._gemm(self.xn, w["w_qkv"], M, H, self.qkv_n, s)
        L.tfd_tree_qkv_append(
            ptr(self.part), sl, M, self.HQ, self.HKV, self.D, ptr(w["gamma_q"]),
            ptr(w["gamma_k"]), ptr(e.cos), ptr(e.sin), e.cap, ptr(pos), ptr(slot), ptr(self.seq),
            table, self.max_pages, ptr(e.kpool[i]), ptr(e.vpool[i]), self.num_pages, self.scale,
            self.eps, ptr(self.q), ptr(e.err), s)
        a = _lib.TfdTreeAttnArgs(
            ptr(self.q), self.nodes * self.QD, self.QD, self.D, ptr(e.kpool[i]), ptr(e.vpool[i]),
            table, ptr(lengths), ptr(counts), ptr(masks), e.B, self.nodes, self.HQ, self.HKV,
            self.D, self.max_pages, self.num_pages, 1.0, ptr(self.attn), 1, ptr(self.attn_work),
            self.attn_work.numel(), ptr(e.err))
        L.tfd_tree_attn(ctypes.addressof(a), s)
        sl = self._gemm(self.attn, w["w_o"], M, self.QD, H, s)
        L.tfd_panel_add_norm(ptr(self.part), sl, ptr(self.hid), ptr(self.h1),
                             ptr(w["gamma_post"]), ptr(self.xn), M, H, self.eps, s)
        self._gate_up(w, M, s)
        sl = self._gemm(self.hmid, w["w_down"], M, I, H, s)
        gamma = self.layers[i + 1]["gamma_in"] if i + 1 < self.L else e.gamma_final
        L.tfd_panel_add_norm(ptr(self.part), sl, ptr(self.h1), ptr(self.hid), ptr(gamma),
                             ptr(self.xn), M, H, self.eps, s)

    def picks_of(self, tokens, parents, counts, lengths) -> torch.Tensor:
        """Greedy picks int32 ``[B, nodes]`` behind every node; the nodes' keys and values stay at
        ``lengths[b] + t`` of the cache."""
        L, e, H = self._lib, self.e, self.H
        M = tokens.numel()
        s = torch.cuda.current_stream(self.dev).cuda_stream
        masks, depths = tree.ancestors(parents, counts, e.err)
        slot = lengths.unsqueeze(1) + self.at
        slot = torch.where(self.at < counts.unsqueeze(1), slot, -1).view(-1)
        pos = (lengths.unsqueeze(1) + depths).view(-1)
        ids = tokens.view(-1).long()
        L.tfd_embed_rows_bf16(ptr(e.w_embed), ptr(ids), ptr(self.hid), H, M, H, e.V, ptr(e.err),
                              s)
        L.tfd_panel_add_norm(None, 0, ptr(self.hid), None, ptr(self.layers[0]["gamma_in"]),
                             ptr(self.xn), M, H, self.eps, s)
        for i in range(self.L):
            self._node_layer(i, M, pos, slot, lengths, counts, masks, s)
        for m in range(0, M, 32):                    # a panel of rows at a time through the head
            L.tfd_gemm_skinny_bf16(ptr(self.xn) + 2 * m * H, ptr(e.w_head), min(32, M - m), H, e.V,
                                   _lib.EPI_LOGITS, None, 0, ptr(self.logits) + 4 * m * e.V, e.V,
                                   ptr(self.work), self.work.numel(), s)
        L.tfd_argmax_rows(ptr(self.logits), e.V, M, e.V, ptr(self.picks), ptr(self.arg_work), s)
        return self.picks


class Speculated:
    """Per-sequence continuations, their timing, and how far the draft carried."""

    def __init__(self, tokens, seconds, prefill_seconds, passes):
        self.tokens: list[list[int]] = tokens
        self.seconds = seconds
        self.prefill_seconds = prefill_seconds
        self.passes = passes                         # model passes, each of all sequences

    @property
    def tokens_per_second(self) -> float:
        n = sum(len(t) for t in self.tokens)
        return n / self.seconds if self.seconds > 0 else float("inf")


class Speculation:
    """Greedy decoding by checked drafts on a batch engine (a weak reference to it)."""

    @staticmethod
    def check(e, nodes: int):
        if not 1 <= nodes <= tree.MAX_NODES:
            raise ValueError(f"nodes must lie in 1..{tree.MAX_NODES}, got {nodes}")
        if e.B * nodes > MAX_PASS:
            raise ValueError(f"{nodes} nodes of {e.B} sequences exceed a pass of {MAX_PASS} rows")

    def __init__(self, engine, nodes: int):
        e = engine()
        self.check(e, nodes)
        self._engine, self.nodes = engine, nodes
        self.step = TreePass(engine, nodes)
        self.cache = Pages([e.kpool, e.vpool], table=e.page_table)
        # what a pass reads: tokens, parents and, in the first place of a row, its nodes
        self.rows = torch.zeros(3, e.B, nodes, dtype=I32, device=e.device)
        self.lengths = torch.zeros(e.B, dtype=I32, device=e.device)
        self.graph = self.found = None

    def _pass(self) -> torch.Tensor:
        """One pass over ``rows``: each sequence's path, how many it holds and the token behind."""
        tokens, parents, counts = self.rows.unbind(0)
        counts = counts[:, 0].contiguous()
        picks = self.step.picks_of(tokens, parents, counts, self.lengths)
        path, accepted, after = tree.accept(tokens, parents, picks, counts)
        self.lengths.copy_(self.cache.keep(self.lengths, path, accepted))
        return torch.cat((path, accepted.unsqueeze(1), after.unsqueeze(1)), 1)

    def _capture(self):
        torch.cuda.synchronize(self._engine().device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.found = self._pass()
        self.graph = graph

    def run(self, prompts, max_new: int, draft) -> Speculated:
        e, T = self._engine(), self.nodes
        prompts = _checked(e, prompts, e.B, max_new)
        if self.graph is None and e.graph is not None:
            self._capture()
        torch.cuda.synchronize(e.device)
        t0 = perf_counter()
        e.prefill(prompts)
        torch.cuda.synchronize(e.device)
        t1 = perf_counter()
        history = [p.tolist() for p in prompts]
        start = [len(p) for p in prompts]
        self.lengths.copy_(e.pos)
        passes = 0
        while True:
            # a draft reaches no further than what is still wanted (node 0 gives one token too)
            left = [max_new - (len(h) - n) for h, n in zip(history, start)]
            if max(left) <= 0:
                break
            rows = np.zeros((3, e.B, T), dtype=np.int32)
            rows[1] = -1
            for b, h in enumerate(history):
                if left[b] <= 0:
                    continue
                tokens, parents = draft(h, min(T, left[b]))
                n = len(tokens)
                if not 1 <= n <= min(T, left[b]) or n != len(parents) or tokens[0] != h[-1]:
                    raise ValueError(f"draft: {n} tokens and {len(parents)} parents, up to "
                                     f"{min(T, left[b])} are wanted, the sequence's last one first")
                if parents[0] != -1 or not all(0 <= p < t for t, p in enumerate(parents[1:], 1)):
                    raise ValueError(f"draft: node 0 has parent -1, every other one a node before "
                                     f"it, got {list(parents)}")
                if not in_vocab(np.asarray(tokens, dtype=np.int64), e.V):
                    raise ValueError(f"draft: token ids must lie in [0, {e.V})")
                rows[0, b, :n], rows[1, b, :n], rows[2, b, 0] = tokens, parents, n
            self.rows.copy_(torch.from_numpy(rows))
            if self.graph is not None:
                self.graph.replay()
                found = self.found
            else:
                found = self._pass()
            passes += 1
            for b, r in enumerate(found.tolist()):
                n = r[T]
                history[b] += [int(rows[0, b, t]) for t in r[1:n]] + ([r[T + 1]] if n else [])
        t2 = perf_counter()
        e.check_errors()
        self.cache.check_errors()
        tokens = [h[n:n + max_new] for h, n in zip(history, start)]
        return Speculated(tokens, t2 - t1, t1 - t0, passes)
