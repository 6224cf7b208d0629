"""``run.py``'s searches: the argument rules, and both on the GPU against its greedy run."""
import pytest

import run as R
from tilefoundry_amd.qwen3.search import NgramDraft

BASE = ["--synthetic", "c1", "--random-prompt", "4", "--max-new-tokens", "4"]


@pytest.mark.parametrize("more", [
    ["--beams", "33"], ["--beams", "-1"], ["--draft", "257"], ["--beams", "2", "--draft", "2"],
    ["--beams", "2", "--sample"], ["--draft", "2", "--sample"], ["--eos", "3"],
    ["--length-penalty", "1"], ["--beams", "2", "--mode", "graph"],
    ["--draft", "2", "--model", "granite"]])
def test_argument_rules(more):
    with pytest.raises(SystemExit):
        R.main(BASE + more)


def test_ngram_draft():
    """The latest continuation of the longest run that came before, branches as one tree."""
    d = NgramDraft(longest=3, branches=2)
    h = [1, 2, 3, 4, 1, 2, 3, 5, 9, 1, 2, 3]
    assert d(h, 8) == ([3, 5, 9, 1, 2, 4, 1, 2], [-1, 0, 1, 2, 3, 0, 5, 6])
    assert d(h, 1) == ([3], [-1]) and d(h, 2) == ([3, 5], [-1, 0])
    assert d([7], 8) == ([7], [-1]) and d([1, 2], 8) == ([2], [-1])
    assert NgramDraft(2, 1)([7, 7, 7], 4) == ([7, 7], [-1, 0])
    # continuations that begin alike share their beginning
    assert d([1, 2, 5, 1, 2, 6, 1], 8) == ([1, 2, 6, 1, 5, 1, 2], [-1, 0, 1, 2, 1, 4, 5])
    for bad in ((0, 1), (1, 0)):
        with pytest.raises(ValueError):
            NgramDraft(*bad)


@pytest.mark.gpu
def test_searches_from_the_command_line(gpu_device, capsys):
    outs = []
    for more in ([], ["--draft", "6"], ["--beams", "1"]):
        assert R.main(["--synthetic", "c1", "--random-prompt", "12", "--max-new-tokens", "12",
                       "--device", gpu_device, "--prefill", *more]) == 0
        outs.append(capsys.readouterr().out)
    assert "6 drafted" in outs[1] and "1 beams" in outs[2]
    assert len(outs[1].splitlines()[0].split()) == 12
