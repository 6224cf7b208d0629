"""Drafted trees, beams, states and pages on the CPU: the definitions the GPU tests compare
with, against hand-worked values, and every refusal that needs no GPU."""
import ctypes
import math

import pytest
import torch

from tests import _search_ref as R
from tilefoundry_amd import _lib, beam, pages, tree
from tilefoundry_amd._lib import TFDError, lib

BF, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
PTR = 1 << 20                       # a well-aligned address that nothing reads


# ------------------------------------------------------------- the definitions
def test_reference_tree():
    p = torch.tensor([[-1, 0, 0, 1, 3, -1]])
    sets, depths = R.ancestors(p)
    assert sets[0] == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 3, 4}, {5}]
    assert depths[0] == [0, 1, 1, 2, 3, 0]
    assert R.words(sets, 6)[0, :, 0].tolist() == [1, 3, 5, 11, 27, 32]
    assert R.words([[{63}, {64}]], 65 - 63).shape == (1, 2, 1)
    tokens = torch.tensor([[9, 4, 5, 6, 6, 9]])
    path, n, after = R.accept(tokens, p, torch.tensor([[4, 6, 0, 2, 0, 0]]))
    assert path.tolist() == [[0, 1, 3, -1, -1, -1]] and n.tolist() == [3]
    assert after.tolist() == [2]
    path, n, after = R.accept(tokens, p, torch.tensor([[7] * 6]), counts=[0])
    assert n.tolist() == [0] and after.tolist() == [-1] and (path == -1).all()


def test_reference_attention():
    """One key: its value.  Two equal keys: their values' mean.  None: zeros."""
    k = torch.zeros(2, 1, 16, 64)
    v = torch.randn(2, 1, 16, 64, generator=torch.Generator().manual_seed(0))
    q = torch.zeros(1, 3, 1, 64)
    table = torch.tensor([[1, 0]])
    masks = torch.tensor([[[1], [3], [0]]])
    out, _ = R.attention(q, k, v, table, [0], masks)
    assert torch.allclose(out[0, 0, 0], v[1, 0, 0].double())
    assert torch.allclose(out[0, 1, 0], v[1, 0, :2].double().mean(0))
    assert not out[0, 2].any()


def test_reference_beam():
    x = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7]]))
    s = torch.tensor([[0.0, -1.0]])
    parents, tokens, scores, lengths, done = R.beam(x, s, None, None, eos=1)
    assert parents.tolist() == [[0, 1]] and tokens.tolist() == [[0, 2]]
    assert torch.allclose(scores, torch.tensor([[math.log(0.5), -1 + math.log(0.7)]]).double())
    assert lengths.tolist() == [[1, 1]] and not done.any()
    # a finished beam stays, and ties go to the lower row and token
    parents, tokens, _, lengths, done = R.beam(
        torch.zeros(2, 3), s, torch.tensor([[4, 4]]), torch.tensor([[False, True]]), eos=1)
    assert parents.tolist() == [[1, 0]] and tokens.tolist() == [[1, 0]]
    assert lengths.tolist() == [[4, 5]] and done.tolist() == [[True, False]]
    # by their means the longer one wins
    got = R.beam(torch.zeros(2, 2), torch.tensor([[-3.0, -1.8]]), torch.tensor([[9, 2]]),
                 torch.tensor([[True, True]]), eos=1, penalty=1.0)
    assert got[0].tolist() == [[0, 1]]
    got = R.beam(torch.full((1, 4), -math.inf), torch.zeros(1, 1), None, None)
    assert got[1].tolist() == [[-1]] and got[2].tolist() == [[-math.inf]]


def test_reference_cache():
    """A row forked in the middle of a page: shared until one of the two writes."""
    pool = torch.zeros(5, 1, 16, 4)
    c = R.Cache([pool], torch.full((2, 3), -1), torch.zeros(5, dtype=I32))
    c.take([0, 0], torch.tensor([20, 0]))
    assert c.table.tolist() == [[0, 1, -1], [-1, -1, -1]] and c.refs.tolist() == [1, 1, 0, 0, 0]
    pool[1, 0, :4] = 7.0
    lengths = c.fork([0, 0], torch.tensor([20, 0]))
    assert lengths.tolist() == [20, 20] and c.refs.tolist() == [2, 2, 0, 0, 0]
    c.take(lengths, 1)
    assert c.table.tolist() == [[0, 1, -1], [0, 2, -1]] and c.refs.tolist() == [2, 1, 1, 0, 0]
    assert pool[2, 0, :4].eq(7).all()
    c.free(torch.tensor([True, False]))
    assert c.refs.tolist() == [1, 0, 1, 0, 0] and c.compact() == 2
    assert c.table.tolist() == [[-1] * 3, [0, 1, -1]] and pool[1, 0, :4].eq(7).all()
    pool[1, 0] = torch.arange(16.0).unsqueeze(1)
    out = c.keep(torch.tensor([0, 18]), torch.tensor([[0, 0, 0], [1, 2, -1]]), [0, 2])
    assert out.tolist() == [0, 20] and pool[1, 0, :6, 0].tolist() == [0, 1, 3, 4, 4, 5]
    assert not c.failed
    c.keep(torch.tensor([0, 18]), torch.tensor([[0, 0, 0], [1, 1, 5]]), [0, 2])
    assert c.failed


# ------------------------------------------------------------------- refusals
def _attention_args(**change):
    a = {"q": torch.zeros(2, 3, 4, 64, dtype=BF), "k_pool": torch.zeros(5, 2, 16, 64, dtype=BF),
         "v_pool": torch.zeros(5, 2, 16, 64, dtype=BF), "table": torch.zeros(2, 2, dtype=I32),
         "lengths": torch.zeros(2, dtype=I32), "masks": torch.zeros(2, 3, 1, dtype=I64)}
    return {**a, **change}


@pytest.mark.parametrize("change,match", [
    ({"q": torch.zeros(2, 3, 4, 64)}, "dtype"), ({"q": torch.zeros(2, 3, 64, dtype=BF)}, "nodes"),
    ({"q": torch.zeros(2, 3, 4, 96, dtype=BF)}, "pools"),
    ({"q": torch.zeros(2, 3, 3, 64, dtype=BF)}, "heads"),
    ({"q": torch.zeros(2, 257, 4, 64, dtype=BF)}, "nodes"),
    ({"q": torch.zeros(2, 0, 4, 64, dtype=BF)}, "nodes"),
    ({"q": torch.zeros(2, 3, 1, 64, dtype=BF)}, "heads"),
    ({"k_pool": torch.zeros(5, 2, 8, 64, dtype=BF)}, "pools"),
    ({"v_pool": torch.zeros(5, 1, 16, 64, dtype=BF)}, "pools"),
    ({"k_pool": torch.zeros(5, 2, 16, 128, dtype=BF)[..., ::2]}, "contiguous"),
    ({"table": torch.zeros(1, 2, dtype=I32)}, "table"),
    ({"table": torch.zeros(2, 0, dtype=I32)}, "table"),
    ({"table": torch.zeros(2, 2, dtype=I64)}, "dtype"),
    ({"lengths": torch.zeros(3, dtype=I32)}, "lengths"),
    ({"masks": torch.zeros(2, 3, 2, dtype=I64)}, "masks"),
    ({"masks": torch.zeros(2, 3, 1, dtype=I32)}, "dtype"),
    ({"scale": 0.0}, "scale"), ({"scale": math.inf}, "scale"), ({"scale": math.nan}, "scale"),
    ({}, "GPU")])
def test_attention_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        tree.attention(**_attention_args(**change))


def test_attention_refuses_head_dims_and_gradients():
    pool = torch.zeros(5, 2, 16, 96, dtype=BF)
    with pytest.raises(ValueError, match="head dimension 96"):
        tree.attention(**_attention_args(q=torch.zeros(2, 3, 4, 96, dtype=BF), k_pool=pool,
                                         v_pool=pool))
    with pytest.raises(ValueError, match="gradients"):
        tree.attention(**_attention_args(q=torch.zeros(2, 3, 4, 64, dtype=BF,
                                                       requires_grad=True)))
    with pytest.raises(TypeError):
        tree.attention(**_attention_args(q=None))


@pytest.mark.parametrize("parents", [
    torch.zeros(2, 3), torch.zeros(3, dtype=I32), torch.zeros(2, 0, dtype=I32),
    torch.zeros(2, 257, dtype=I32), torch.zeros(65536, 1, dtype=I32),
    torch.zeros(2, 3, dtype=I32)])
def test_ancestors_and_accept_refuse(parents):
    with pytest.raises(ValueError):
        tree.ancestors(parents)
    with pytest.raises(ValueError):
        tree.accept(parents, parents, parents)


def test_accept_refuses_unlike_shapes():
    a, b = torch.zeros(2, 3, dtype=I32), torch.zeros(2, 4, dtype=I32)
    with pytest.raises(ValueError, match="picks"):
        tree.accept(a, a, b)
    with pytest.raises(ValueError, match="parents"):
        tree.accept(a, b, a)


@pytest.mark.parametrize("kw", [
    {"beams": 0}, {"beams": 65}, {"beams": 4, "eos": -1}, {"beams": 4, "eos": 1 << 20},
    {"beams": 4, "length_penalty": -0.1}, {"beams": 4, "length_penalty": math.nan},
    {"beams": 4, "length_penalty": 101.0}])
def test_beam_rules_refuse(kw):
    with pytest.raises(ValueError):
        beam.Beam(**kw)


@pytest.mark.parametrize("change,match", [
    ({"logits": torch.zeros(8, 50, dtype=torch.float64)}, "dtype"),
    ({"logits": torch.zeros(7, 50)}, "logits"), ({"logits": torch.zeros(8, 0)}, "vocabulary"),
    ({"logits": torch.zeros(8, 9)}, "vocabulary"), ({"scores": torch.zeros(8)}, "scores"),
    ({"scores": torch.zeros(4, 2)}, "scores"), ({"scores": torch.zeros(2, 4, dtype=BF)}, "dtype"),
    ({"lengths": torch.zeros(2, 4)}, "dtype"), ({"lengths": torch.zeros(8, dtype=I32)}, "lengths"),
    ({"done": torch.zeros(2, 4)}, "dtype"),
    ({"done": torch.zeros(4, 2, dtype=torch.bool)}, "done"), ({}, "GPU")])
def test_beam_refuses(change, match):
    a = {"logits": torch.zeros(8, 50), "scores": torch.zeros(2, 4), **change}
    with pytest.raises(ValueError, match=match):
        beam.Beam(4, eos=11)(**a)


def test_states_refuse():
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="no tensors"):
        beam.States([])
    with pytest.raises(TypeError):
        beam.States([x, 3])
    for other in (torch.zeros(3, 6), torch.zeros(()), torch.zeros(6, 4).t()):
        with pytest.raises(ValueError, match="contiguous"):
            beam.States([x, other])
    with pytest.raises(ValueError, match="GPU"):
        beam.States([x])


@pytest.mark.parametrize("pools,kw,match", [
    ([], {}, "no pools"), ([torch.zeros(4, 2, 8, 16)], {}, "contiguous pools"),
    ([torch.zeros(4, 16, 16)], {}, "contiguous pools"),
    ([torch.zeros(4, 2, 16, 16).transpose(0, 1)], {}, "contiguous pools"),
    ([torch.zeros(0, 4, 2, 16, 16)], {}, "layers"), ([torch.zeros(4, 2, 16, 16)], {}, "GPU")])
def test_pages_refuse(pools, kw, match):
    with pytest.raises(ValueError, match=match):
        pages.Pages(pools, rows=2, max_pages=2, **kw)


# --------------------------------------------------------------- the C entries
def _refused(entry, args, code, match):
    with pytest.raises(TFDError, match=match) as e:
        getattr(lib(), entry)(ctypes.addressof(args) if isinstance(args, ctypes.Structure)
                              else args, 0)
    assert e.value.code == code


def _tree_args(**kw):
    a = {"q": PTR, "q_row": 512, "q_node": 256, "q_head": 64, "k_pool": PTR, "v_pool": PTR,
         "page_table": PTR, "lengths": PTR, "masks": PTR, "rows": 2, "nodes": 2, "heads": 4,
         "kv_heads": 2, "head_dim": 64, "max_pages": 4, "num_pages": 9, "scale": 1.0, "out": PTR}
    return _lib.TfdTreeAttnArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,code,match", [
    ({"nodes": 0}, -2, "nodes=0"), ({"nodes": 257}, -2, "nodes"), ({"heads": 3}, -2, "heads"),
    ({"head_dim": 80}, -2, "head_dim"), ({"max_pages": 0}, -2, "max_pages"),
    ({"num_pages": 0}, -2, "num_pages"), ({"rows": -1}, -2, "rows"),
    ({"scale": 0.0}, -1, "scale"), ({"scale": math.nan}, -1, "scale"), ({"q": 0}, -1, "null"),
    ({"out": 0}, -1, "null"), ({"q": PTR + 2}, -1, "aligned"), ({"q_head": 68}, -1, "aligned"),
    ({"k_pool": PTR + 8}, -1, "aligned"), ({"out": PTR + 8}, -1, "aligned"),
    ({"max_pages": 4000}, -1, "work"),
    ({"max_pages": 4000, "work": PTR, "work_bytes": 16}, -1, "work")])
def test_tree_attn_entry_refuses(kw, code, match):
    _refused("tfd_tree_attn", _tree_args(**kw), code, match)


def test_tree_attn_work():
    L = lib()
    assert L.tfd_tree_attn_work_bytes(1, 4, 4, 2, 64, 4) >= 0
    assert L.tfd_tree_attn_work_bytes(1, 4, 4, 2, 64, 4000) > 0
    for bad in [(1, 4, 4, 2, 96, 4000), (1, 0, 4, 2, 64, 4000), (0, 4, 4, 2, 64, 4000),
                (1, 4, 5, 2, 64, 4000)]:
        assert L.tfd_tree_attn_work_bytes(*bad) == 0
    assert L.tfd_tree_attn(ctypes.addressof(_tree_args(rows=0)), 0) == 0


def _beam_args(**kw):
    a = {"logits": PTR, "ldl": 100, "type": _lib.TYPE_F32, "scores": PTR, "groups": 2, "beams": 4,
         "vocab": 100, "eos": 3, "parents": PTR, "tokens": PTR, "scores_out": PTR,
         "lengths_out": PTR, "done_out": PTR, "work": PTR, "work_bytes": 1 << 20}
    return _lib.TfdBeamArgs(**{**a, **kw})


@pytest.mark.parametrize("kw,code,match", [
    ({"type": 3}, -1, "type"), ({"beams": 0}, -2, "beams"), ({"beams": 65}, -2, "beams"),
    ({"vocab": 0}, -2, "vocab"), ({"vocab": 1 << 21}, -2, "vocab"), ({"groups": 65536}, -2, "groups"),
    ({"groups": 65535, "beams": 64, "vocab": 100000, "ldl": 100000}, -2, "groups"),
    ({"eos": 100}, -1, "eos"), ({"eos": -2}, -1, "eos"), ({"penalty": -1.0}, -1, "penalty"),
    ({"penalty": math.nan}, -1, "penalty"), ({"logits": 0}, -1, "null"),
    ({"done_out": 0}, -1, "null"), ({"ldl": 99}, -1, "ldl"), ({"logits": PTR + 2}, -1, "ldl"),
    ({"work": 0}, -1, "work"), ({"work_bytes": 8}, -1, "work"), ({"work": PTR + 8}, -1, "work")])
def test_beam_entry_refuses(kw, code, match):
    _refused("tfd_beam_select", _beam_args(**kw), code, match)


def test_beam_work_and_empty_calls():
    L = lib()
    assert L.tfd_beam_work_bytes(2, 4, 100) > 0 and L.tfd_beam_work_bytes(2, 65, 100) == 0
    assert L.tfd_beam_select(ctypes.addressof(_beam_args(groups=0)), 0) == 0
    assert L.tfd_reorder_states(PTR, 0, 0, PTR, 1, 4, 0, 0) == 0
    assert L.tfd_state_blocks(PTR, 4096) == 1 and L.tfd_state_blocks(PTR, 4097) == 5
    assert L.tfd_state_blocks(PTR, 0) == 0
    for bad in [(PTR, -1, 0, PTR, 1, 4), (PTR, 1, 1, PTR, 1, 65), (PTR, 1, 1, PTR, 1, 0),
                (PTR, 1, 1 << 24, PTR, 1, 4), (0, 1, 1, PTR, 1, 4),
                (PTR, 1, 1, 0, 1, 4)]:
        with pytest.raises(TFDError):
            L.tfd_reorder_states(*bad, 0, 0)


@pytest.mark.parametrize("at,value", [(0, 0), (1, 0), (2, -1), (3, 3), (4, 0), (5, 100), (6, 0),
                                      (11, 0), (12, 0), (13, 0), (14, 0), (15, 0), (16, 0),
                                      (18, 0), (21, 0)])
def test_tree_qkv_append_refuses(at, value):
    args = [PTR, 1, 4, 4, 2, 64, PTR, PTR, PTR, PTR, 64, PTR, PTR, PTR, PTR, 4, PTR, PTR, 8, 1.0,
            1e-6, PTR, 0, 0]
    args[at] = value
    with pytest.raises(TFDError):
        lib().tfd_tree_qkv_append(*args)


def test_tree_entries_refuse():
    L = lib()
    assert L.tfd_tree_masks(0, 0, 0, 5, 0, 0, 0, 0) == 0
    assert L.tfd_tree_accept(0, 0, 0, 0, 0, 5, 0, 0, 0, 0) == 0
    for rows, nodes in ((-1, 4), (2, 0), (2, 257)):
        with pytest.raises(TFDError):
            L.tfd_tree_masks(PTR, 0, rows, nodes, PTR, PTR, 0, 0)
        with pytest.raises(TFDError):
            L.tfd_tree_accept(PTR, PTR, PTR, 0, rows, nodes, PTR, PTR, PTR, 0)
    with pytest.raises(TFDError):
        L.tfd_tree_masks(0, 0, 2, 4, PTR, PTR, 0, 0)
    with pytest.raises(TFDError):
        L.tfd_tree_accept(PTR, PTR, PTR, 0, 2, 4, 0, PTR, PTR, 0)


def _pages_args(**kw):
    a = {"pools": PTR, "n_pools": 2, "max_page_bytes": 4096, "table": PTR, "refs": PTR, "rows": 2,
         "max_pages": 3, "num_pages": 9, "scratch": PTR}
    return _lib.TfdPages(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    {"rows": 0}, {"rows": 1025}, {"max_pages": 0}, {"num_pages": 0}, {"n_pools": -1},
    {"max_page_bytes": -1}, {"table": 0}, {"refs": 0}, {"scratch": 0}, {"pools": 0},
    {"rows": 1024, "max_pages": 1 << 22}])
def test_pages_entries_refuse(kw):
    L, at = lib(), _pages_args(**kw)
    p = ctypes.addressof(at)
    for call in (lambda: L.tfd_pages_fork(p, PTR, 0, PTR, PTR, 0),
                 lambda: L.tfd_pages_take(p, PTR, 0, 1, 0),
                 lambda: L.tfd_pages_copy(p, PTR, PTR, 1, 0),
                 lambda: L.tfd_pages_keep(p, PTR, PTR, PTR, 4, PTR, 0),
                 lambda: L.tfd_pages_compact(p, PTR, 0)):
        with pytest.raises(TFDError):
            call()


def test_pages_entries_refuse_null_lists():
    L, at = lib(), _pages_args()
    p = ctypes.addressof(at)
    for call in (lambda: L.tfd_pages_fork(p, PTR, 0, 0, PTR, 0),
                 lambda: L.tfd_pages_fork(p, 0, 0, 0, 0, 0),
                 lambda: L.tfd_pages_take(p, 0, 0, 1, 0),
                 lambda: L.tfd_pages_copy(p, 0, PTR, 1, 0),
                 lambda: L.tfd_pages_copy(p, PTR, PTR, -1, 0),
                 lambda: L.tfd_pages_keep(p, PTR, 0, PTR, 4, PTR, 0),
                 lambda: L.tfd_pages_keep(p, PTR, PTR, PTR, 0, PTR, 0),
                 lambda: L.tfd_pages_keep(ctypes.addressof(_pages_args(n_pools=0)), PTR, PTR, PTR,
                                          4, PTR, 0)):
        with pytest.raises(TFDError):
            call()
    assert L.tfd_pages_copy(p, PTR, PTR, 0, 0) == 0


def test_structs_and_constants_match_the_header(tmp_path):
    import re
    import shutil
    import subprocess
    from pathlib import Path

    header = Path(__file__).resolve().parent.parent / "include" / "tf_search.h"
    defines = dict(re.findall(r"^#define TFD_(\w+) (\d+)", header.read_text(), re.M))
    for name in ("ERR_ROW_RANGE", "ERR_NO_PAGES", "TREE_MAX_NODES", "BEAM_MAX", "BEAM_MAX_VOCAB",
                 "PAGES_MAX_ROWS"):
        assert getattr(_lib, name) == int(defines[name]), name
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    structs = (_lib.TfdTreeAttnArgs, _lib.TfdBeamArgs, _lib.TfdState, _lib.TfdPool, _lib.TfdPages)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"',
             "int main(void) {"]
    want = []
    for cls in structs:
        name = cls.__name__
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    lines.append('  printf("%lld\\n", (long long)TFD_PAGES_SCRATCH(7, 11, 100));')
    want.append(_lib.pages_scratch(7, 11, 100))
    (tmp_path / "probe.c").write_text("\n".join(lines + ["  return 0; }"]))
    subprocess.run(["gcc", str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True)
    assert [int(v) for v in out.stdout.split()] == want


def test_tensors_that_share_memory_are_refused():
    """What one block of a call moves another would move again."""
    x = torch.zeros(6, 2, 16, 16)
    whole = torch.zeros(3, 6, 2, 16, 16)
    for pools in ([x, x], [x, x.view(6, 1, 32, 16)[:, :, :16].contiguous(), x.view(6, 2, 16, 16)],
                  [whole, whole[1]], [whole[:2], whole[1:]]):
        with pytest.raises(ValueError, match="overlap"):
            pages.Pages(pools, rows=2, max_pages=2)
        with pytest.raises(ValueError, match="overlap|one number"):
            beam.States(pools)
    with pytest.raises(ValueError, match="GPU"):     # (side by side, or nothing in them)
        pages.Pages([whole[0], whole[1], x], rows=2, max_pages=2)
    with pytest.raises(ValueError, match="GPU"):
        beam.States([x, x[:, :0], x[:, :0], torch.zeros_like(x)])
