"""The measured cases' ranges, on the CPU: what a drawn case asks of the framework's handles."""
import random

import pytest
import torch

from perf import more_operators as cases
from tilefoundry_amd import _lib, beam


@pytest.mark.parametrize("first", [0, 2000])
def test_reordering_cases_move_within_their_groups(monkeypatch, first):
    """Every listed and drawn reordering is made in groups of its beams, which divide its rows and
    fit one call."""
    made = []
    monkeypatch.setattr(beam, "States", lambda tensors, beams=None: made.append((tensors, beams)))
    monkeypatch.setitem(cases.MAKE, "reorder", lambda case, seed: {
        "states": [torch.zeros(case["groups"] * case["beams"], 1)]})
    monkeypatch.setattr(cases, "own", True)
    wanted = [cases.draw(random.Random(s)) for s in range(first, first + 2000)] + cases.listed()
    wanted = [c for c in wanted if c["kind"] == "reorder"]
    for case in wanted:
        cases.prepare(case, 1)
        tensors, beams = made.pop()
        assert beams == case["beams"] and 1 <= beams <= _lib.BEAM_MAX
        assert tensors[0].shape[0] % beams == 0
    assert len(wanted) > 200
