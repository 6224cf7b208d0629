"""Microscaled tensors and the experts' choice on the CPU: the definitions the GPU tests
compare with, against hand-worked values, and every refusal that needs no GPU."""
import ctypes
import math

import pytest
import torch

from tests import _mx4_ref as R
from tilefoundry_amd import _lib, mx4, routing
from tilefoundry_amd._lib import TFDError, lib

BF = torch.bfloat16
PTR = 1 << 20                       # a well-aligned address that nothing reads


def test_reference_grid_ties_and_scales():
    """Ties between neighbours go to the even code; the scale follows the largest."""
    x = torch.zeros(1, 32)
    x[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    codes, scales = R.quantise(x)
    assert scales.tolist() == [[127]]
    got = R.values(codes, scales)[0, :8].tolist()
    assert got == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    tiny = torch.full((1, 32), 2.0 ** -140)
    assert R.quantise(tiny)[1].item() == 0
    bad = torch.zeros(1, 64)
    bad[0, 3] = math.inf
    assert R.quantise(bad)[1].tolist() == [[255, 0]]
    # half a step is the most a value in range is off by
    y = torch.randn(8, 64, dtype=torch.float64)
    v = R.values(*R.quantise(y)).reshape(-1, 32)
    top = y.reshape(-1, 32).abs().amax(1, keepdim=True)
    scale = 2.0 ** (torch.floor(torch.log2(top)) - 2)
    inside = y.reshape(-1, 32).abs() <= 6 * scale
    assert ((v - y.reshape(-1, 32)).abs() <= scale + 1e-12)[inside].all()


def test_reference_route_masks_and_groups():
    logits = torch.tensor([[0.0, 5.0, -math.inf, math.nan, 1.0, 1.0]])
    w, ids = R.route(logits, None, k=4, score="sigmoid", shared=1)
    assert ids.tolist() == [[1, 4, 5, 0, 6]] and w[0, -1] == 1
    w, ids = R.route(logits, None, k=2, score="softmax", groups=3, keep=1)
    assert ids.tolist() == [[4, 5]] or ids.tolist() == [[1, 0]]
    w, ids = R.route(torch.full((1, 4), -math.inf), None, k=2, score="softmax")
    assert ids.tolist() == [[-1, -1]] and w.tolist() == [[0.0, 0.0]]


def test_mx4_tensor_refuses_what_does_not_fit():
    c, s = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8)
    t = mx4.Mx4(c, s)
    assert t.shape == (3, 64) and t[1].shape == (64,) and t[0:2].shape == (2, 64)
    for codes, scales in [(c.int(), s), (c, s[:2]), (c, s[:, :1]), (c[:, :0], s[:, :0])]:
        with pytest.raises(ValueError):
            mx4.Mx4(codes, scales)
    with pytest.raises(IndexError):
        t[1][0]
    with pytest.raises(ValueError, match="dtype"):
        t.dequantise(torch.float64)
    with pytest.raises(ValueError, match="GPU"):
        t.dequantise()


@pytest.mark.parametrize("x,match", [
    (torch.zeros(2, 33), "multiple of 32"), (torch.zeros(2, 0), "multiple of 32"),
    (torch.zeros(()), "multiple of 32"), (torch.zeros(2, 32, dtype=torch.float64), "dtype"),
    (torch.zeros(2, 32, requires_grad=True), "gradients"), (torch.zeros(2, 32), "GPU")])
def test_quantise_refuses(x, match):
    with pytest.raises(ValueError, match=match):
        mx4.quantise(x)


@pytest.mark.parametrize("kwargs", [
    dict(top_k=0), dict(top_k=65), dict(top_k=60, shared=5), dict(top_k=2, shared=-1),
    dict(top_k=2, score="tanh"), dict(top_k=2, groups=4, kept_groups=5),
    dict(top_k=2, groups=0), dict(top_k=2, kept_groups=0), dict(top_k=2, group_top=3),
    dict(top_k=2, scale=0.0), dict(top_k=2, scale=math.inf), dict(top_k=2, scale=math.nan)])
def test_routing_refuses_settings(kwargs):
    with pytest.raises(ValueError):
        routing.Routing(**kwargs)


@pytest.mark.parametrize("logits,bias,match", [
    (torch.zeros(4), None, "rows, experts"), (torch.zeros(2, 513), None, "experts"),
    (torch.zeros(2, 30), None, "multiple"), (torch.zeros(2, 4), None, "top_k"),
    (torch.zeros(2, 32, dtype=torch.float64), None, "dtype"),
    (torch.zeros(2, 32), torch.zeros(31), "bias"),
    (torch.zeros(2, 32), torch.zeros(32, dtype=BF), "dtype"),
    (torch.zeros(2, 32, requires_grad=True), None, "gradients"),
    (torch.zeros(2, 32), None, "GPU")])
def test_routing_refuses_inputs(logits, bias, match):
    with pytest.raises(ValueError, match=match):
        routing.Routing(top_k=4, groups=4, kept_groups=2)(logits, bias)


def test_quantise_entries_refuse():
    """What the kernels would read or write wrongly is refused before a launch."""
    L = lib()

    def quantise(x=PTR, ldx=64, type=0, rows=4, K=64, codes=PTR, ldc=32, scales=PTR, lds=2):
        return L.tfd_mx4_quantise(x, ldx, type, rows, K, codes, ldc, scales, lds, None)

    def dequantise(codes=PTR, ldc=32, scales=PTR, lds=2, rows=4, K=64, out=PTR, ldo=64, type=1):
        return L.tfd_mx4_dequantise(codes, ldc, scales, lds, rows, K, out, ldo, type, None)

    def pack(codes=PTR, scales=PTR, codes2=None, scales2=None, N=16, K=64, packed=PTR):
        return L.tfd_mx4_pack(codes, scales, codes2, scales2, N, K, packed, None)

    for call in [lambda: quantise(K=33), lambda: quantise(K=0), lambda: quantise(rows=-1),
                 lambda: quantise(x=None), lambda: quantise(codes=None),
                 lambda: quantise(ldx=63), lambda: quantise(ldc=33), lambda: quantise(ldc=28),
                 lambda: quantise(lds=1), lambda: quantise(type=3), lambda: quantise(x=PTR + 1),
                 lambda: quantise(codes=PTR + 2),
                 lambda: dequantise(K=48), lambda: dequantise(out=None),
                 lambda: dequantise(ldo=65), lambda: dequantise(ldo=62),
                 lambda: dequantise(type=-1), lambda: dequantise(out=PTR + 2),
                 lambda: pack(K=31), lambda: pack(N=0), lambda: pack(packed=None),
                 lambda: pack(codes2=PTR), lambda: pack(codes=PTR + 8)]:
        with pytest.raises(TFDError):
            call()
    assert quantise(rows=0) == 0 and dequantise(rows=0) == 0
    assert L.tfd_mx4_packed_bytes(17, 160) == 2 * (2 * 1024 + 256)
    assert L.tfd_mx4_packed_bytes(0, 160) == 0 and L.tfd_mx4_packed_bytes(16, 33) == 0


@pytest.mark.parametrize("K", [32, 64, 8192])
def test_quantise_entries_refuse_launches_of_too_many_threads(K):
    """A thread has eight values, and a launch's threads, in whole blocks of 256, 32 bits."""
    L = lib()
    first = (2 ** 32 - 256) // (K // 8) + 1
    for rows in (first, 2 ** 32 // (K // 8), 2 ** 40):
        with pytest.raises(TFDError, match="mx4_quantise"):
            L.tfd_mx4_quantise(PTR, K, 1, rows, K, PTR, K // 2, PTR, K // 32, None)
        with pytest.raises(TFDError, match="mx4_dequantise"):
            L.tfd_mx4_dequantise(PTR, K // 2, PTR, K // 32, rows, K, PTR, K, 1, None)
    tiles = (2 ** 32 - 256) // (-(-K // 512) * 256) + 1
    for N in (tiles * 16, 2 ** 62):
        with pytest.raises(TFDError, match="mx4_pack"):
            L.tfd_mx4_pack(PTR, PTR, None, None, N, K, PTR, None)
        with pytest.raises(TFDError, match="mx4_pack"):
            L.tfd_mx4_pack(PTR, PTR, PTR, PTR, N, K, PTR, None)


def test_route_entry_refuses():
    def call(**over):
        f = dict(logits=PTR, ldl=32, type=0, bias=None, rows=2, experts=32, k=4, score=0,
                 groups=4, kept_groups=2, group_top=2, shared=1, renormalise=1, scale=1.0,
                 weights=PTR, ids=PTR, ld=5)
        f.update(over)
        return lib().tfd_route_experts(ctypes.addressof(_lib.TfdRouteArgs(**f)), None)

    for bad in [dict(logits=None), dict(weights=None), dict(ids=None), dict(type=5),
                dict(score=2), dict(experts=513), dict(experts=0), dict(rows=-1), dict(groups=3),
                dict(groups=0), dict(kept_groups=5), dict(kept_groups=0), dict(group_top=0),
                dict(k=0), dict(k=17), dict(k=65, kept_groups=4, experts=512),
                dict(shared=-1), dict(shared=62), dict(scale=0.0), dict(scale=math.inf),
                dict(scale=math.nan), dict(ldl=31), dict(ld=4), dict(logits=PTR + 2),
                dict(bias=PTR + 1)]:
        with pytest.raises(TFDError):
            call(**bad)
    with pytest.raises(TFDError):
        lib().tfd_route_experts(None, None)
    assert call(rows=0) == 0


class _NoGpu:
    """Handles as their methods see them, without a GPU to pack weights on."""

    @staticmethod
    def linear(N, K):
        lin = object.__new__(mx4.Linear)
        lin.N, lin.K, lin.device, lin.index, lin.packed = N, K, torch.device("cuda:0"), 0, None
        return lin

    @staticmethod
    def experts(E, H, I):
        ex = object.__new__(mx4.Experts)
        ex.E, ex.H, ex.I, ex.device, ex.index = E, H, I, torch.device("cuda:0"), 0
        return ex


def _mx(*shape):
    return mx4.Mx4(torch.zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8),
                   torch.zeros(*shape[:-1], shape[-1] // 32, dtype=torch.uint8))


def test_linear_refuses():
    for w in (_mx(64), _mx(2, 3, 64)):
        with pytest.raises(ValueError, match="N, K"):
            mx4.Linear(w)
    with pytest.raises(ValueError, match="GPU"):
        mx4.Linear(_mx(3, 64))
    lin = _NoGpu.linear(3, 64)
    for x, kw, match in [(torch.zeros(2, 64), {}, "dtype"),
                         (torch.zeros(2, 32, dtype=BF), {}, "weights"),
                         (torch.zeros(2, 64, dtype=BF), dict(dtype=torch.float16), "dtype"),
                         (torch.zeros((), dtype=BF), {}, "dimensions"),
                         (torch.zeros(2, 64, dtype=BF, requires_grad=True), {}, "gradients"),
                         (torch.zeros(2, 64, dtype=BF), {}, "on cpu"), (_mx(2, 64), {}, "on cpu"),
                         (_mx(2, 32), {}, "weights")]:
        with pytest.raises(ValueError, match=match):
            lin(x, **kw)
    with pytest.raises(TypeError):
        lin([1.0])


def test_experts_refuse():
    for shapes in [((2, 32, 64), (2, 32, 64), (2, 32, 64)), ((2, 32, 64), (2, 64, 64), (2, 64, 32)),
                   ((32, 64), (32, 64), (64, 32)), ((513, 32, 32),) * 3]:
        with pytest.raises(ValueError, match="Experts"):
            mx4.Experts(*[_mx(*s) for s in shapes])
    with pytest.raises(ValueError, match="GPU"):
        mx4.Experts(_mx(2, 32, 64), _mx(2, 32, 64), _mx(2, 64, 32))
    ex = _NoGpu.experts(4, 64, 32)
    x, ids, w = torch.zeros(3, 64, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for bad in [(x.float(), ids, w), (x, ids.long(), w), (x, ids, w.to(BF)), (x[:, :32], ids, w),
                (x[0], ids, w), (x, ids[:2], w), (x, ids, w[:, :1]), (x, ids[:, :0], w[:, :0]),
                (x, ids, w.clone().requires_grad_()), (x, ids, w)]:
        with pytest.raises(ValueError):
            ex(*bad)
    with pytest.raises(ValueError, match="dtype"):
        ex(x, ids, w, dtype=torch.float16)


def test_product_entries_refuse():
    def gemm(**over):
        f = dict(x=PTR, ldx=64, x_scales=None, ldxs=0, w=PTR, M=4, K=64, N=10, out=PTR, ldo=10,
                 out_type=1)
        f.update(over)
        return lib().tfd_mx4_gemm(ctypes.addressof(_lib.TfdMx4GemmArgs(**f)), None)

    for bad in [dict(x=None), dict(w=None), dict(out=None), dict(K=48), dict(K=0), dict(N=0),
                dict(M=-1), dict(ldx=56), dict(ldx=68), dict(ldo=9), dict(out_type=2),
                dict(x=PTR + 8), dict(w=PTR + 4), dict(out=PTR + 1),
                dict(x_scales=PTR, ldx=16, ldxs=2), dict(x_scales=PTR, ldx=32, ldxs=1),
                dict(x_scales=PTR, ldx=40, ldxs=2)]:
        with pytest.raises(TFDError):
            gemm(**bad)
    with pytest.raises(TFDError):
        lib().tfd_mx4_gemm(None, None)
    assert gemm(M=0) == 0

    need = lib().tfd_mx4_experts_work_bytes(40, 2, 4, 64, 32)

    def experts(**over):
        f = dict(x=PTR, ldx=64, ids=PTR, weights=PTR, ld=2, w_gu=PTR, w_down=PTR, rows=40, k=2,
                 experts=4, H=64, I=32, out=PTR, ldo=64, out_type=1, accumulate=0, mult=1.0,
                 work=PTR, work_bytes=need, err=None)
        f.update(over)
        return lib().tfd_mx4_experts(ctypes.addressof(_lib.TfdMx4ExpertsArgs(**f)), None)

    for bad in [dict(x=None), dict(ids=None), dict(weights=None), dict(w_gu=None),
                dict(w_down=None), dict(out=None), dict(work=None), dict(H=48), dict(I=0),
                dict(rows=-1), dict(rows=65536), dict(k=0), dict(k=65), dict(experts=0),
                dict(experts=513), dict(ldx=56), dict(ldx=65), dict(ld=1), dict(ldo=63),
                dict(out_type=2), dict(x=PTR + 2), dict(work=PTR + 16), dict(ids=PTR + 2),
                dict(work_bytes=need - 1), dict(out=PTR + 1)]:
        with pytest.raises(TFDError):
            experts(**bad)
    with pytest.raises(TFDError):
        lib().tfd_mx4_experts(None, None)
    assert experts(rows=0) == 0
    # a step of few rows needs the hidden values alone, as two bf16
    assert lib().tfd_mx4_experts_work_bytes(16, 8, 4, 64, 32) == 16 * 8 * 32 * 4
    assert lib().tfd_mx4_experts_work_bytes(0, 8, 4, 64, 32) == 0
    # a list: 51 hidden rows, 51 f32 outputs, 4 words, 8 tiles of 4 words and the order
    assert lib().tfd_mx4_experts_work_bytes(17, 3, 8, 64, 64) == 6656 + 13056 + 512


def test_structs_match_c_layout(tmp_path):
    """The ctypes structures of include/tf_mx4.h have the C compiler's layout."""
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    structs = {n: getattr(_lib, n) for n in ("TfdRouteArgs", "TfdMx4GemmArgs",
                                             "TfdMx4ExpertsArgs")}
    header = Path(__file__).resolve().parent.parent / "include" / "tf_mx4.h"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"',
             "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({name}));')
        lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join([*lines, "  return 0; }"]))
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    want = []
    for cls in structs.values():
        want += [ctypes.sizeof(cls), *[getattr(cls, f).offset for f, _ in cls._fields_]]
    assert got == want
    text = header.read_text()
    for name in ("TYPE_F32", "TYPE_BF16", "TYPE_F16", "SCORE_SOFTMAX", "SCORE_SIGMOID",
                 "ROUTE_MAX_EXPERTS"):
        assert f"#define TFD_{name} {getattr(_lib, name)}\n" in text


def test_run_takes_4_bit_experts_for_granite_alone():
    import run

    for synthetic in ("c1", "c2", "c4"):
        with pytest.raises(SystemExit, match="granite"):
            run.main(["--synthetic", synthetic, "--random-prompt", "4", "--experts", "mx4"])


@pytest.mark.parametrize("E,k,H,I", [(72, 12, 4096, 768), (256, 8, 2048, 512),
                                     (14, 12, 1024, 4096), (8, 4, 64, 512), (512, 2, 32, 32),
                                     (512, 1, 32, 32), (3, 64, 32, 4096), (1, 1, 4096, 32)])
def test_experts_workspace_covers_fewer_rows(E, k, H, I):
    """A workspace of `rows` rows serves every call of fewer, which may run in another way:
    what the entry asks for never falls as rows grow.  (The prompt passes keep one for their
    largest.)"""
    need = lib().tfd_mx4_experts_work_bytes
    sizes = [need(m, k, E, H, I) for m in range(1, 65536)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def _far(*shape, dtype=torch.float32):
    """One element seen as a tensor of that shape: sizes without the memory."""
    return torch.zeros(1, dtype=dtype).expand(*shape)


PAST = 2 ** 32 + 32                 # 32 where 32 bits are kept


def test_sizes_past_32_bits_are_refused():
    """Dimensions that the C entries take as 32-bit integers: cut to those they would name a
    smaller tensor, of which the kernels would compute a part and leave the rest unwritten."""
    u8 = torch.uint8

    def far(*shape):
        return mx4.Mx4(_far(*shape[:-1], shape[-1] // 2, dtype=u8),
                       _far(*shape[:-1], shape[-1] // 32, dtype=u8))

    for K in (2 ** 31, PAST):
        with pytest.raises(ValueError, match="last dimension"):
            mx4.quantise(_far(1, K))
        with pytest.raises(ValueError, match="last dimension"):
            far(1, K).dequantise()
    for N, K in ((16, PAST), (PAST, 32), (2 ** 24 + 1, 32), (16, 2 ** 22 + 32)):
        with pytest.raises(ValueError, match="Linear: weights of up to"):
            mx4.Linear(far(N, K))
    for H, I in ((PAST, 32), (32, PAST), (2 ** 20 + 32, 32), (32, 2 ** 20 + 32)):
        with pytest.raises(ValueError, match="Experts: hidden and width"):
            mx4.Experts(far(2, I, H), far(2, I, H), far(2, H, I))


def test_routing_refuses_rows_past_a_launch():
    """Four rows a block of 256 threads, and a launch's threads have 32 bits; from 2^32 rows
    on an integer of the entry would hold the rest of them."""
    most = 4 * ((2 ** 32 - 256) // 256)
    rule = routing.Routing(top_k=1)
    for rows in (most + 1, 2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ValueError, match=f"up to {most} rows"):
            rule(_far(rows, 2))
    with pytest.raises(ValueError, match="GPU"):
        rule(_far(most, 2))
    for rows in (most + 1, 2 ** 31 - 1):
        a = _lib.TfdRouteArgs(logits=PTR, ldl=2, rows=rows, experts=2, k=1, groups=1,
                              kept_groups=1, group_top=2, scale=1.0, weights=PTR, ids=PTR, ld=1)
        with pytest.raises(TFDError, match="rows="):
            lib().tfd_route_experts(ctypes.addressof(a), None)


def test_forward_mode_inputs_are_refused():
    """A tangent would be dropped without a word; a detached input, or no_grad with a plain
    one, is taken as far as the device's check."""
    from torch.autograd import forward_ad

    rule = routing.Routing(top_k=2)
    ex, ids = _NoGpu.experts(4, 64, 32), torch.zeros(3, 2, dtype=torch.int32)
    x, w = torch.zeros(3, 64), torch.zeros(3, 2)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in [lambda: mx4.quantise(dual(x)), lambda: _NoGpu.linear(3, 64)(dual(x.to(BF))),
                     lambda: rule(dual(x)), lambda: rule(x, dual(torch.zeros(64))),
                     lambda: ex(dual(x.to(BF)), ids, w), lambda: ex(x.to(BF), ids, dual(w))]:
            with pytest.raises(ValueError, match="gradients"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradients"):
                call()
        with pytest.raises(ValueError, match="GPU"):
            mx4.quantise(dual(x).detach())
        with pytest.raises(ValueError, match="GPU"):
            mx4.quantise(x)
    with pytest.raises(ValueError, match="gradients"):
        torch.func.jvp(mx4.quantise, (x,), (x,))


def test_reference_route_ranks_groups_by_their_best_two():
    """(0, 5) outranks (1, 1), and the masked pair has nothing: the first group, best first."""
    logits = torch.tensor([[0.0, 5.0, -math.inf, math.nan, 1.0, 1.0]])
    assert R.route(logits, None, k=2, score="softmax", groups=3, keep=1)[1].tolist() == [[1, 0]]


def _form(M, K, N, both=False):
    form = (ctypes.c_int32 * 4)()
    lib().tfd_mx4_gemm_form(int(both), M, K, N, form)
    return list(form)


def test_products_of_few_rows_have_no_work():
    """mx4.Linear asks for work past MX4_WHOLE_ROWS alone: up to there K is never split, and the
    header's number is the package's."""
    from pathlib import Path

    header = Path(__file__).resolve().parent.parent / "include" / "tf_mx4.h"
    assert f"#define TFD_MX4_WHOLE_ROWS {_lib.MX4_WHOLE_ROWS}\n" in header.read_text()
    work = lib().tfd_mx4_gemm_work_bytes
    for M in (1, 16, 17, 33, _lib.MX4_WHOLE_ROWS):
        for K in (32, 544, 2048, 6144, 65536, 1 << 22):
            for N in (1, 17, 2048, 12288, 1 << 20):
                assert work(M, K, N) == 0
                assert _form(M, K, N)[2] == _form(M, K, N, True)[2] == 1
    for M, K, N in ((65, 1184, 130), (66, 2176, 70), (128, 6144, 260), (300, 4128, 513)):
        parts = max(_form(M, K, N)[2], _form(M, K, N, True)[2])
        assert parts > 1 and work(M, K, N) == parts * M * (-(-N // 4) * 4) * 4


def test_form_entries_refuse():
    form = (ctypes.c_int32 * 4)()
    for M, K, N in ((0, 64, 64), (-1, 64, 64), (4, 48, 64), (4, 0, 64), (4, 64, 0),
                    (4, 64, 2 ** 24 + 1), (4, 2 ** 22 + 32, 64)):
        with pytest.raises(TFDError):
            lib().tfd_mx4_gemm_form(0, M, K, N, form)
    with pytest.raises(TFDError):
        lib().tfd_mx4_gemm_form(0, 4, 64, 64, None)
    tile = lib().tfd_mx4_experts_tile_rows
    for bad in ((0, 1, 1, 32, 32), (65536, 1, 1, 32, 32), (1, 0, 1, 32, 32), (1, 65, 1, 32, 32),
                (1, 1, 0, 32, 32), (1, 1, 513, 32, 32), (1, 1, 1, 0, 32), (1, 1, 1, 32, 0)):
        assert tile(*bad) == -1
    assert tile(16, 8, 64, 64, 32) == 0 and tile(16, 9, 64, 64, 32) != 0
