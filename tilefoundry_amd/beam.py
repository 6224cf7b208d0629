"""Beam search over logits on the device, and the states that follow the beams.

``Beam`` holds a search's rule and is called with one step's logits: of all beams' next tokens it
keeps the best, by their log probabilities' sum, divided by ``length ** length_penalty``.

    beam = Beam(beams=4, eos=2, length_penalty=0.6)
    step = beam(logits, scores, lengths, done)       # logits [groups * beams, vocab]
    states.reorder(step.parents)                     # States: each row becomes its parent's
    lengths_in_cache = cache.fork(step.parents.view(-1), lengths_in_cache)   # pages.Pages

A group is one sequence's beams, row ``group * beams + beam``.  At a search's start one beam of
a group has score 0 and the others minus infinity, which offer nothing.  The exact
definitions are declared in ``include/tf_search.h``.

Every call runs on its tensors' device and that device's current stream, allocates its outputs
like any torch operation (so calls can be captured into a HIP graph and made from several
streams) and computes no gradients.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import lib, ptr
from .mx4 import (FLOAT32, INT32, TYPES, _settle, check_apart, check_device, check_input, launch,
                  row_stride, rows_of)

BOOL = (torch.bool, torch.uint8)
MAX_GROUPS = 65535


class Step(NamedTuple):
    """One step's beams, each ``[groups, beams]``, the best first."""

    parents: torch.Tensor       # int32: the row that each continues
    tokens: torch.Tensor        # int32, -1 for a place that no candidate was left for
    scores: torch.Tensor        # f32: sums of log probabilities
    lengths: torch.Tensor       # int32
    done: torch.Tensor          # bool


@dataclass(frozen=True)
class Beam:
    """A search's rule; see the module docstring.

    ``eos``: the token that finishes a beam (None: none does).  A finished beam stays as it is and
    competes with its own score and length.  ``length_penalty``: 0 compares the sums, 1 their
    means."""

    beams: int
    eos: int | None = None
    length_penalty: float = 0.0

    def __post_init__(self):
        if not 1 <= self.beams <= _lib.BEAM_MAX:
            raise ValueError(f"beams must lie in 1..{_lib.BEAM_MAX}, got {self.beams}")
        if self.eos is not None and not 0 <= self.eos < _lib.BEAM_MAX_VOCAB:
            raise ValueError(f"eos must be a token, got {self.eos}")
        if not 0 <= self.length_penalty <= 100:
            raise ValueError(f"length_penalty must lie in 0..100, got {self.length_penalty}")

    def __call__(self, logits: torch.Tensor, scores: torch.Tensor,
                 lengths: torch.Tensor | None = None,
                 done: torch.Tensor | None = None) -> Step:
        """Logits ``[groups * beams, vocab]`` (f32, bf16 or f16) and the beams' scores f32,
        lengths int32 (None: zeros) and done bool (None: none), ``[groups, beams]``."""
        check_input(logits, "logits", TYPES)
        check_input(scores, "scores", FLOAT32)
        if scores.dim() != 2 or scores.shape[1] != self.beams:
            raise ValueError(f"scores must be [groups, {self.beams}], got {tuple(scores.shape)}")
        groups, K = scores.shape
        if logits.dim() != 2 or logits.shape[0] != groups * K:
            raise ValueError(f"logits must be [{groups * K}, vocab], got {tuple(logits.shape)}")
        vocab = logits.shape[1]
        if not 1 <= vocab <= _lib.BEAM_MAX_VOCAB or (self.eos is not None and self.eos >= vocab):
            raise ValueError(f"a vocabulary of 1 to {_lib.BEAM_MAX_VOCAB} with eos {self.eos} in "
                             f"it, got {vocab}")
        if groups > MAX_GROUPS or groups * K * -(-vocab // 1024) >= 1 << 23:
            raise ValueError(f"{groups} groups of {K} beams over {vocab} tokens are too many for "
                             "one call")
        for t, what, types in ((lengths, "lengths", INT32), (done, "done", BOOL)):
            if t is not None:
                check_input(t, what, types)
                if t.shape != scores.shape:
                    raise ValueError(f"{what} must be {tuple(scores.shape)}, got "
                                     f"{tuple(t.shape)}")
        check_device(logits.device, scores, lengths, done)
        logits, scores = rows_of(logits), scores.contiguous()
        lengths = None if lengths is None else lengths.contiguous()
        done = None if done is None else done.contiguous()
        parents, tokens, length, score = scores.new_empty((4, groups, K),
                                                          dtype=torch.int32).unbind(0)
        score = score.view(torch.float32)
        over = scores.new_empty((groups, K), dtype=torch.bool)
        L = lib()
        need = L.tfd_beam_work_bytes(groups, K, vocab)
        # of the stream that uses it, like the outputs
        work = scores.new_empty(need, dtype=torch.uint8)
        a = _lib.TfdBeamArgs(
            ptr(logits), row_stride(logits), TYPES[logits.dtype], ptr(scores), ptr(lengths),
            ptr(done), groups, K, vocab, -1 if self.eos is None else self.eos,
            self.length_penalty, ptr(parents), ptr(tokens), ptr(score), ptr(length), ptr(over),
            ptr(work), need)
        launch(logits.get_device(), L.tfd_beam_select, ctypes.addressof(a))
        return Step(parents, tokens, score, length, over)


class States:
    """Tensors whose rows follow the beams: recurrent states, conv windows, token histories.

    Each is contiguous ``[rows, ...]`` of any type, all of one number of rows, on one GPU, no two
    in the same memory; they are kept.  Rows move within groups of *beams* (default: all rows, up to 64)."""

    def __init__(self, tensors, beams: int | None = None):
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("States: no tensors")
        first = self.tensors[0]
        for t in self.tensors:
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"States: expected tensors, got {type(t).__name__}")
            check_input(t, "States", (t.dtype,))
            if t.dim() < 1 or t.shape[0] != first.shape[0] or not t.is_contiguous():
                raise ValueError(f"States: contiguous tensors of one number of rows, got "
                                 f"{tuple(t.shape)} beside {tuple(first.shape)}")
        check_apart(self.tensors, "States")
        check_device(first.device, *self.tensors)
        self.rows, self.device = first.shape[0], first.device
        self.beams = beams if beams is not None else self.rows
        if not 1 <= self.beams <= _lib.BEAM_MAX or self.rows % self.beams:
            raise ValueError(f"States: groups of 1..{_lib.BEAM_MAX} rows that divide "
                             f"{self.rows}, got {self.beams}")
        if self.rows // self.beams > MAX_GROUPS:
            raise ValueError(f"States: up to {MAX_GROUPS} groups, got {self.rows // self.beams}")
        L, blocks, entries = lib(), 0, []
        sizes = [t.numel() // self.rows * t.element_size() for t in self.tensors]
        for t, size in zip(self.tensors, sizes):
            if size:
                entries.append(_lib.TfdState(ptr(t), size, blocks))
                blocks += L.tfd_state_blocks(ptr(t), size)
        if blocks >= 1 << 24:
            raise ValueError("States: rows of up to 64 GiB in all")
        self.blocks, self.n = blocks, len(entries)
        raw = bytes((_lib.TfdState * len(entries))(*entries)) or b"\0"
        self._entries = torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(self.device)
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.index = self.err.get_device()
        _settle(self.device)

    def reorder(self, parents: torch.Tensor) -> None:
        """Row r of every tensor becomes what row ``parents[r]`` was (int32, ``[rows]`` or
        ``[groups, beams]``), in place.  A parent outside the row's group leaves the row as it is
        and makes ``check_errors`` raise."""
        check_input(parents, "parents", INT32)
        if parents.numel() != self.rows or parents.dim() > 2 or \
                (parents.dim() == 2 and parents.shape[1] != self.beams):
            raise ValueError(f"parents must be [{self.rows}], got {tuple(parents.shape)}")
        if parents.get_device() != self.index:
            raise ValueError(f"States: parents on {parents.device}, tensors on {self.device}")
        parents = parents.contiguous()
        launch(self.index, lib().tfd_reorder_states, ptr(self._entries), self.n, self.blocks,
               ptr(parents), self.rows // self.beams, self.beams, ptr(self.err))

    def check_errors(self) -> None:
        """Raises if a call since the last check met a parent outside its row's group (waits
        for the device)."""
        torch.cuda.synchronize(self.device)
        if int(self.err.item()):
            self.err.zero_()
            torch.cuda.synchronize(self.device)
            raise RuntimeError("States: a parent outside its row's group was skipped")
