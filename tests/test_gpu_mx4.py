"""Microscaled 4-bit kernels against their definitions in 64 bits.

Quantisation is exact: codes and scales are compared bit for bit.  Products: a bf16 or f32
output is off by its one rounding (finfo.eps / 2 of the value) and by the f32 sums, which
are bounded by K roundings of 2^-24 of the sum of magnitudes.
"""
import math

import pytest
import torch

from tests import _mx4_ref as R
from tilefoundry_amd import mx4

pytestmark = pytest.mark.gpu

BF, F32, F16, F64 = torch.bfloat16, torch.float32, torch.float16, torch.float64


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _hard_rows(K, seed):
    """Rows that meet every rounding: ties, signs, zeros, extremes of the scales, values
    that are not finite."""
    g = _gen(seed)
    ties = torch.randint(-64, 65, (6, K), generator=g) / 8.0
    rows = [torch.randn(8, K, generator=g), ties, ties * 2.0 ** -20,
            torch.randn(2, K, generator=g) * 2.0 ** -124, torch.zeros(1, K), -torch.zeros(1, K),
            torch.full((1, K), 2.0 ** -149), torch.full((1, K), 3e38),
            torch.randn(2, K, generator=g) * 2.0 ** -140]
    x = torch.cat(rows)
    bad = torch.randn(3, K, generator=g)
    bad[0, 0], bad[1, K - 1], bad[2, K // 2] = math.inf, -math.inf, math.nan
    return torch.cat((x, bad))


@pytest.mark.parametrize("K", [32, 96, 256, 4128])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_quantise_bit_for_bit(gpu_device, dtype, K):
    x = _hard_rows(K, K).to(dtype)
    got = mx4.quantise(x.to(gpu_device))
    codes, scales = R.quantise(x)
    assert torch.equal(got.scales.cpu(), scales)
    assert torch.equal(got.codes.cpu(), codes)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_dequantise_every_code_and_scale(gpu_device, dtype):
    """All 256 scales x 16 codes; past the type's range an infinity, as the value rounds."""
    scales = torch.arange(256, dtype=torch.uint8).unsqueeze(1)
    all_codes = torch.randint(0, 256, (256, 16), dtype=torch.uint8, generator=_gen(0))
    all_codes[:, :8] = torch.tensor([0x10, 0x32, 0x54, 0x76, 0x98, 0xba, 0xdc, 0xfe],
                                    dtype=torch.uint8)
    t = mx4.Mx4(all_codes.to(gpu_device), scales.to(gpu_device))
    got, want = t.dequantise(dtype).cpu(), R.values(all_codes, scales).to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf),
                       want.nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf))


def test_quantise_strides_and_shapes(gpu_device):
    """Sliced, padded, transposed, broadcast and empty inputs give what a copy gives."""
    base = torch.randn(9, 3, 200, generator=_gen(1)).to(gpu_device)
    for x in [base[:, 1, 8:200], base[:, :, 3:131], base[::2, :, :192], base[0, 0, 1:65],
              base[:0, 0, :96],
              base[:, :, :32].transpose(0, 1), base[0, :1, :64].expand(5, 64),
              torch.randn(64, 7, generator=_gen(2)).to(gpu_device).t()]:
        got, want = mx4.quantise(x), mx4.quantise(x.clone(memory_format=torch.contiguous_format))
        assert got.shape == tuple(x.shape)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    t = mx4.quantise(base[:, :, :192])
    part = t[2:7, 1]
    assert torch.equal(part.dequantise(), t.dequantise()[2:7, 1])


def test_quantise_large_and_replayed(gpu_device):
    """More rows than one pass of blocks, and a captured call on new inputs."""
    x = torch.randn(20000, 64, generator=_gen(3)).to(gpu_device)
    q = mx4.quantise(x)
    codes, scales = R.quantise(x[-40:])
    assert torch.equal(q.codes[-40:].cpu(), codes) and torch.equal(q.scales[-40:].cpu(), scales)
    static = x[:100].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mx4.quantise(static).dequantise(BF)
    for i in range(3):
        static.copy_(x[200 * i:200 * i + 100])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, mx4.quantise(static).dequantise(BF))


# ------------------------------------------------------------------ projections
def _weights(rows, K, seed, scale=0.05):
    w = torch.randn(rows, K, generator=_gen(seed)) * scale
    return mx4.Mx4(*R.quantise(w)) if rows * K <= 1 << 16 else _gpu_weights(w)


def _gpu_weights(w):
    """Quantised by the kernel that test_quantise_bit_for_bit checks (the CPU's loop over
    blocks takes long at these sizes)."""
    q = mx4.quantise(w.to("cuda:0"))
    return mx4.Mx4(q.codes.cpu(), q.scales.cpu())


def _to(t, dev):
    return mx4.Mx4(t.codes.to(dev), t.scales.to(dev))


def _check_product(got, x64, w64):
    """Half a step of the output type, and 2 K roundings of 2^-24 of the magnitudes' sum
    (one for each product added, one for the matrix cores' order).  A sum whose magnitudes
    add up to s may hold any value up to s on its way: where s reaches the f32 range
    (2^128 - 2^104) an order of adding exists that passes it, so nothing is asked there."""
    want, size = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    within = size < torch.finfo(F32).max
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + 2 * x64.shape[1] * 2.0 ** -24 * size
    bad = within & ~((got.cpu().to(F64) - want).abs() <= bound * 1.01 + 1e-300)
    assert not bad.any(), (bad.nonzero()[:4], got.cpu()[bad][:4], want[bad][:4])


@pytest.mark.parametrize("M,K,N", [
    (1, 32, 1), (1, 2048, 64), (2, 96, 17), (15, 480, 130), (16, 512, 48), (17, 160, 100),
    (32, 128, 16), (33, 1184, 70), (64, 256, 33), (65, 224, 260), (128, 544, 64),
    (129, 96, 19), (300, 1024, 321), (1, 32, 2000), (5, 8192, 31), (257, 32, 15)])
@pytest.mark.parametrize("both", [False, True])
def test_linear(gpu_device, M, K, N, both):
    w = _weights(N, K, M + N)
    x = torch.randn(M, K, generator=_gen(K)).to(BF)
    lin = mx4.Linear(_to(w, gpu_device))
    if both:
        q = mx4.Mx4(*R.quantise(x)) if M * K <= 1 << 16 else _gpu_weights(x)
        given, x64 = _to(q, gpu_device), R.values(q.codes, q.scales)
    else:
        given, x64 = x.to(gpu_device), x.to(F64)
    w64 = R.values(w.codes, w.scales)
    for dtype in (BF, F32):
        _check_product(lin(given, dtype=dtype), x64, w64)


@pytest.mark.parametrize("M", [3, 40, 150])
def test_linear_rows_stay_apart(gpu_device, M):
    """A row that is not finite changes no other row; values beyond K (a padded input's) are
    not read, whatever they are; extreme scales come through."""
    K, N = 160, 50
    w = _weights(N, K, 1)
    w.scales[4] = 255                                  # output 4 is NaN
    w.scales[7, :] = 1                                 # 2^-126
    w.scales[9, :] = 250
    lin = mx4.Linear(_to(w, gpu_device))
    base = torch.full((M, 256), math.nan, dtype=BF)
    base[:, 8:8 + K] = torch.randn(M, K, generator=_gen(2)).to(BF)
    base[1, 8 + 37] = math.inf
    base[2, 8 + 140] = math.nan
    x = base.to(gpu_device)[:, 8:8 + K]
    got = lin(x, dtype=F32)
    assert got[:, 4].isnan().all() and got[2].isnan().all()
    assert not got[1].isfinite().any()
    rows = [m for m in range(M) if m not in (1, 2)]
    cols = [n for n in range(N) if n != 4]
    x64, w64 = base[:, 8:8 + K].to(F64), R.values(w.codes, w.scales)
    _check_product(got[rows][:, cols], x64[rows], w64[cols])
    q = mx4.quantise(x)                                # the block becomes NaN, its row with it
    got = lin(q, dtype=F32)
    assert got[1].isnan().all() and got[2].isnan().all()
    v = R.values(q.codes, q.scales)
    _check_product(got[rows][:, cols], v[rows], w64[cols])


def test_linear_strides_shapes_empty(gpu_device):
    lin = mx4.Linear(_to(_weights(40, 96, 3), gpu_device))
    base = torch.randn(6, 5, 200, generator=_gen(4)).to(BF).to(gpu_device)
    for x in [base[:, :, :96], base[:, 2, 1:97], base[::2, :, 100:196], base[0, 0, :96],
              base[:0, 0, :96], base[0, :1, :96].expand(7, 96),
              torch.randn(96, 20, generator=_gen(5)).to(BF).to(gpu_device).t()]:
        want = lin(x.clone(memory_format=torch.contiguous_format))
        got = lin(x)
        assert got.shape == (*x.shape[:-1], 40) and torch.equal(got, want)
    q = mx4.quantise(base[:, :, :96])
    assert torch.equal(lin(q[1:4, 2]), lin(q)[1:4, 2])
    sliced = mx4.Mx4(mx4.quantise(base[:, 0, :192]).codes[:, 48:],
                     mx4.quantise(base[:, 0, :192]).scales[:, 3:])
    assert torch.equal(lin(sliced), lin(mx4.quantise(base[:, 0, 96:192])))


@pytest.mark.parametrize("M", [1, 20, 70])
def test_linear_repeats_and_replays(gpu_device, M):
    """The same bits every time, from a second stream and from a replayed graph."""
    K, N = 2048, 520
    lin = mx4.Linear(_to(_weights(N, K, 6), gpu_device))
    x = torch.randn(4, M, K, generator=_gen(7)).to(BF).to(gpu_device)
    want = [lin(v) for v in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [lin(v) for v in x]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    static = x[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = lin(mx4.quantise(static))
        z = lin(static)
    for i in (1, 2, 3):
        static.copy_(x[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(z, want[i]) and torch.equal(y, lin(mx4.quantise(x[i])))


@pytest.mark.parametrize("M,K,N,both", [(1, 6144, 12288, False), (48, 4096, 8512, False),
                                        (1000, 2048, 6144, False), (700, 4096, 2048, True),
                                        (1024, 1056, 8512, False), (1024, 1056, 8512, True),
                                        (4001, 544, 8500, False), (4001, 544, 8500, True)])
def test_linear_at_model_sizes(gpu_device, M, K, N, both):
    """Every output against 64-bit products on the GPU."""
    w = mx4.quantise((torch.randn(N, K, generator=_gen(8)) * 0.02).to(gpu_device))
    x = torch.randn(M, K, generator=_gen(9)).to(BF).to(gpu_device)
    given = mx4.quantise(x) if both else x
    got = mx4.Linear(w)(given, dtype=F32)
    x64 = given.dequantise().double() if both else x.double()
    wt = w.dequantise().double().t().contiguous()
    want, size = x64 @ wt, x64.abs() @ wt.abs()
    bound = 2.0 ** -24 * want.abs() + 2 * K * 2.0 ** -24 * size
    assert ((got.double() - want).abs() <= bound * 1.01).all()


# ---------------------------------------------------------------------- experts
def _experts(E, H, I, seed, dev):
    parts = [mx4.quantise((torch.randn(E, *s, generator=_gen(seed + i)) * 0.1).to(dev))
             for i, s in enumerate([(I, H), (I, H), (H, I)])]
    return mx4.Experts(*parts), [p.dequantise().double() for p in parts]


def _check_experts(got, x, ids, weights, values, mult=1.0, start=None):
    """Against 64 bits throughout.  Off by: the hidden values' rounding to bf16 (2^-8 of
    each; as two bf16, in calls of up to 16 rows and 128 places, 2^-16), the gate and up sums' f32 roundings through the SiLU (whose slope stays under
    1.1), the down sums', and half a step of the output type."""
    gate, up, down = values
    u = 2.0 ** -24
    two = x.shape[0] <= 16 and ids.numel() <= 128
    hidden = 2.0 ** -16 if two else 2.0 ** -8
    x64 = x.double()
    H, I = x.shape[1], gate.shape[1]
    want = torch.zeros(got.shape, dtype=F64, device=got.device)
    off = torch.zeros_like(want)
    for e in range(gate.shape[0]):
        row, slot = torch.nonzero(ids == e, as_tuple=True)
        if not row.numel():
            continue
        xe = x64[row]
        g, v, d = (t[e].t().contiguous() for t in (gate, up, down))
        a, b = xe @ g, xe @ v
        ea, eb = 2 * H * u * (xe.abs() @ g.abs()), 2 * H * u * (xe.abs() @ v.abs())
        s = a / (1 + torch.exp(-a))
        h = s * b
        eh = 1.1 * ea * b.abs() + s.abs() * eb + ea * eb + h.abs() * (hidden + 16 * u)
        w = weights[row, slot].double().unsqueeze(1)
        y = h @ d
        ey = eh @ d.abs() + 2 * I * u * ((h.abs() + eh) @ d.abs())
        want.index_add_(0, row, y * w)
        off.index_add_(0, row, (ey + 4 * u * (h.abs() @ d.abs())) * w.abs())
    want, off = want * mult, off * abs(mult) * (1 + ids.shape[1] * u)
    if start is not None:
        want = want + start.double()
        off = off + 2 * u * want.abs()
    bound = off + torch.finfo(got.dtype).eps / 2 * (want.abs() + off) + 1e-30
    bad = ~((got.double() - want).abs() <= bound * 1.01)
    assert not bad.any(), (bad.nonzero()[:4], got[bad][:4], want[bad][:4], bound[bad][:4])


def _choice(rows, E, k, seed, dev, empty=0.0, repeat=False):
    g = _gen(seed)
    if repeat:
        ids = torch.randint(0, E, (rows, k), generator=g)
    else:
        ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(rows)]) if rows \
            else torch.zeros(0, k)
    ids = torch.where(torch.rand(rows, k, generator=g) < empty, torch.full_like(ids, -1), ids)
    weights = torch.randn(rows, k, generator=g)
    return ids.to(torch.int32).to(dev), weights.to(dev)


@pytest.mark.parametrize("rows,E,k,H,I", [
    (1, 1, 1, 32, 32), (1, 8, 2, 96, 64), (1, 64, 8, 256, 160), (3, 5, 5, 64, 96),
    (16, 8, 8, 160, 128), (16, 40, 8, 512, 96), (12, 9, 10 - 1, 288, 32), (17, 8, 3, 64, 64),
    (33, 70, 4, 128, 160), (60, 4, 2, 192, 96), (130, 6, 3, 352, 224), (300, 3, 2, 64, 64),
    (400, 2, 2, 96, 32), (2, 64, 64, 64, 32)])
def test_experts(gpu_device, rows, E, k, H, I):
    ex, values = _experts(E, H, I, rows + E, gpu_device)
    x = torch.randn(rows, H, generator=_gen(H)).to(BF).to(gpu_device)
    ids, weights = _choice(rows, E, k, rows, gpu_device)
    for dtype in (BF, F32):
        _check_experts(ex(x, ids, weights, dtype=dtype), x, ids, weights, values)
    ex.check_errors()


@pytest.mark.parametrize("rows", [1, 9, 16, 40, 500])
def test_experts_empty_places_and_repeats(gpu_device, rows):
    """Empty places, rows of nothing else, an expert several times in a row, one expert for
    all rows, one expert for none."""
    E, k, H, I = 7, 6, 64, 96
    ex, values = _experts(E, H, I, 11, gpu_device)
    x = torch.randn(rows, H, generator=_gen(12)).to(BF).to(gpu_device)
    for seed, empty, repeat in [(1, 0.4, False), (2, 0.0, True), (3, 0.7, True)]:
        ids, weights = _choice(rows, E, k, seed, gpu_device, empty, repeat)
        ids[rows // 2] = -1
        _check_experts(ex(x, ids, weights), x, ids, weights, values)
        assert (ex(x, ids, weights)[rows // 2] == 0).all()
    ids, weights = _choice(rows, E, k, 4, gpu_device)
    for only in (0, E - 1):
        ids.fill_(only)
        _check_experts(ex(x, ids, weights), x, ids, weights, values)
    ids.fill_(-1)
    assert (ex(x, ids, weights) == 0).all()
    # as ids come from a router, garbage weights stand beside empty places
    weights.fill_(math.nan)
    assert (ex(x, ids, weights) == 0).all()
    ex.check_errors()


@pytest.mark.parametrize("rows", [2, 16, 100])
def test_experts_bad_ids_are_skipped_and_raise(gpu_device, rows):
    ex, values = _experts(4, 64, 32, 13, gpu_device)
    x = torch.randn(rows, 64, generator=_gen(14)).to(BF).to(gpu_device)
    ids, weights = _choice(rows, 4, 3, 15, gpu_device)
    for bad in (4, -2, 2 ** 31 - 1, -2 ** 31):
        ids[rows - 1, 1] = bad
        _check_experts(ex(x, ids, weights), x, ids, weights, values)
        with pytest.raises(RuntimeError, match="id outside"):
            ex.check_errors()
    ex.check_errors()


@pytest.mark.parametrize("rows", [5, 50, 300])
def test_experts_rows_stay_apart(gpu_device, rows):
    """A row with a value that is not finite, or an overflow in its hidden values, changes no
    other row, those of the same tile included."""
    E, k, H, I = 3, 2, 96, 64
    ex, values = _experts(E, H, I, 16, gpu_device)
    base = torch.full((rows, 160), math.nan, dtype=BF)
    base[:, 16:16 + H] = torch.randn(rows, H, generator=_gen(17)).to(BF)
    base[0, 20], base[3, 30] = math.nan, math.inf
    x = base.to(gpu_device)[:, 16:16 + H]
    ids, weights = _choice(rows, E, k, 18, gpu_device)
    got = ex(x, ids, weights, dtype=F32)
    keep = torch.tensor([r for r in range(rows) if r not in (0, 3)], device=gpu_device)
    assert got[0].isnan().all() and not got[3].isfinite().any()
    _check_experts(got[keep], x[keep], ids[keep], weights[keep], values)


@pytest.mark.parametrize("rows", [4, 60, 300])
def test_experts_accumulate_entry(gpu_device, rows):
    """The C entry on padded rows: out + mult * y into a bf16 and an f32 stream, the padding
    and the rows behind the last left as they were."""
    import ctypes

    from tilefoundry_amd import _lib
    from tilefoundry_amd._lib import lib, ptr

    E, k, H, I = 5, 3, 64, 96
    ex, values = _experts(E, H, I, 19, gpu_device)
    x = torch.randn(rows, H, generator=_gen(20)).to(BF).to(gpu_device)
    ids, weights = _choice(rows, E, k, 21, gpu_device)
    wide_i = torch.full((rows, k + 2), 999, dtype=torch.int32, device=gpu_device)
    wide_w = torch.full((rows, k + 2), math.nan, device=gpu_device)
    wide_i[:, :k], wide_w[:, :k] = ids, weights
    need = lib().tfd_mx4_experts_work_bytes(rows, k, E, H, I)
    work = torch.full((need,), 255, dtype=torch.uint8, device=gpu_device)
    for dtype, kind in ((BF, _lib.TYPE_BF16), (F32, _lib.TYPE_F32)):
        for accumulate in (0, 1):
            out = torch.randn(rows + 2, H + 6, generator=_gen(22)).to(dtype).to(gpu_device)
            before = out.clone()
            a = _lib.TfdMx4ExpertsArgs(ptr(x), H, ptr(wide_i), ptr(wide_w), k + 2, ptr(ex.w_gu),
                                       ptr(ex.w_down), rows, k, E, H, I, ptr(out), H + 6, kind,
                                       accumulate, 0.22, ptr(work), need, None)
            lib().tfd_mx4_experts(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
            _check_experts(out[:rows, :H], x, ids, weights, values, mult=0.22,
                           start=before[:rows, :H] if accumulate else None)
            assert torch.equal(out[rows:], before[rows:])
            assert torch.equal(out[:, H:], before[:, H:])


@pytest.mark.parametrize("rows", [1, 8, 30, 200])
def test_experts_repeat_and_replay(gpu_device, rows):
    """The same bits on every call, on two streams at once and from replayed graphs that
    share the handle; nothing is kept from one call for the next."""
    E, k, H, I = 12, 4, 256, 128
    ex, _ = _experts(E, H, I, 23, gpu_device)
    xs = torch.randn(4, rows, H, generator=_gen(24)).to(BF).to(gpu_device)
    picks = [_choice(rows, E, k, 25 + i, gpu_device) for i in range(4)]
    want = [ex(x, *p) for x, p in zip(xs, picks)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ex(xs[i], *picks[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    graphs = []
    for i in range(2):
        static = [xs[0].clone(), picks[0][0].clone(), picks[0][1].clone()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ex(*static)
        graphs.append((g, static, y))
    for i in (1, 2, 3):
        for g, static, y in graphs:
            for t, v in zip(static, (xs[i], *picks[i])):
                t.copy_(v)
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for _, _, y in graphs)


@pytest.mark.parametrize("rows,E,k,H,I", [(1, 256, 8, 2048, 512), (8, 72, 10, 4096, 768),
                                          (250, 256, 8, 2048, 512), (600, 72, 10, 4096, 768)])
def test_experts_at_model_sizes(gpu_device, rows, E, k, H, I):
    g = torch.Generator(device=gpu_device).manual_seed(rows)
    parts = [mx4.quantise(torch.randn(E, *s, generator=g, device=gpu_device) * 0.02)
             for s in [(I, H), (I, H), (H, I)]]
    ex = mx4.Experts(*parts)
    x = torch.randn(rows, H, generator=g, device=gpu_device).to(BF)
    ids, weights = _choice(rows, E, k, 3, gpu_device)
    _check_experts(ex(x, ids, weights), x, ids, weights,
                   [p.dequantise().double() for p in parts])


def test_serving_chain(gpu_device):
    """Quantise, project, route, experts with a shared one, as a layer runs them -- eagerly
    and as one captured graph, for a prompt and for single tokens."""
    from tilefoundry_amd.routing import Routing

    E, k, H, I, shared = 16, 4, 256, 96, 1
    ex, values = _experts(E + shared, H, I, 30, gpu_device)
    router = _gpu_weights(torch.randn(E, H, generator=_gen(31)) * 0.1)
    lin, rule = mx4.Linear(_to(router, gpu_device)), Routing(
        top_k=k, score="sigmoid", groups=4, kept_groups=2, scale=2.0, shared=shared)
    bias = torch.randn(E, generator=_gen(32)).mul(0.1).to(gpu_device)

    def layer(x):
        logits = lin(x, dtype=F32)
        weights, ids = rule(logits, bias)
        return logits, weights, ids, ex(x, ids, weights)

    for rows in (1, 16, 90):
        x = torch.randn(rows, H, generator=_gen(rows)).to(BF).to(gpu_device)
        logits, weights, ids, y = layer(x)
        _check_product(logits, x.cpu().to(F64), R.values(router.codes, router.scales))
        want_w, want_i = R.route(logits, bias, k=k, score="sigmoid", groups=4, keep=2,
                                 scale=2.0, shared=shared)
        assert torch.equal(ids.cpu(), want_i)
        _check_experts(y, x, ids, weights, values)
        static = torch.zeros_like(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(static)
        for _ in range(3):
            static.copy_(x)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[3], y) and torch.equal(out[2], ids)
            static.zero_()
    ex.check_errors()


@pytest.mark.parametrize("M,K,N", [(17, 6144, 40), (33, 2080, 300), (64, 4096, 129),
                                   (65, 1184, 130), (128, 6144, 260), (500, 544, 70),
                                   (260, 4128, 513)])
@pytest.mark.parametrize("both", [False, True])
def test_linear_parts_of_k(gpu_device, M, K, N, both):
    """Products of more than 64 rows but few blocks add parts of K in a second launch: right
    with the work they ask for and, in one launch, without; the same bits on every call."""
    import ctypes

    from tilefoundry_amd import _lib
    from tilefoundry_amd._lib import lib, ptr

    w = mx4.quantise((torch.randn(N, K, generator=_gen(K)) * 0.05).to(gpu_device))
    x = torch.randn(M, K, generator=_gen(M)).to(BF).to(gpu_device)
    given = mx4.quantise(x) if both else x
    x64 = (given.dequantise() if both else x).double().cpu()
    w64 = w.dequantise().double().cpu()
    lin = mx4.Linear(w)
    if K >= 4096:
        assert M <= 64 or lib().tfd_mx4_gemm_work_bytes(M, K, N) > 0
    for dtype, kind in ((BF, _lib.TYPE_BF16), (F32, _lib.TYPE_F32)):
        got = lin(given, dtype=dtype)
        _check_product(got, x64, w64)
        assert torch.equal(got, lin(given, dtype=dtype))
        out = torch.full((M + 1, N + 3), 7.0, dtype=dtype, device=gpu_device)
        rows, scales = (given.codes, given.scales) if both else (x, None)
        a = _lib.TfdMx4GemmArgs(ptr(rows), rows.shape[1], ptr(scales), K // 32 if both else 0,
                                ptr(lin.packed), M, K, N, ptr(out), N + 3, kind, None, 0)
        lib().tfd_mx4_gemm(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
        _check_product(out[:M, :N], x64, w64)
        assert (out[M:] == 7).all() and (out[:, N:] == 7).all()


# ----------------------------------------------------------- offsets past 32 bits
def test_rows_past_4_gib(gpu_device):
    """Rows whose bytes start past 2^32: quantised, back, and multiplied, with 16, 100 and
    all rows a call; a strided view too."""
    M, K, N = (1 << 22) + 37, 512, 32
    x = torch.zeros(M, K, dtype=BF, device=gpu_device)
    tail = torch.randn(100, K, generator=_gen(40)).to(BF)
    x[-100:] = tail.to(gpu_device)
    q = mx4.quantise(x)
    codes, scales = R.quantise(tail)
    assert torch.equal(q.codes[-100:].cpu(), codes) and torch.equal(q.scales[-100:].cpu(), scales)
    assert not q.codes[:-100].any()
    back = q[-100:].dequantise()
    assert torch.equal(q.dequantise(BF)[-100:].float(), back)
    w = _weights(N, K, 41)
    lin = mx4.Linear(_to(w, gpu_device))
    w64 = R.values(w.codes, w.scales).to(F64)
    for rows in (16, 100, M):
        for t, t64 in ((x, tail.to(F64)), (q, back.cpu().to(F64))):
            n = min(rows, 100)
            _check_product(lin(t[-rows:], dtype=F32)[-n:], t64[-n:], w64)
    # every 65,536th row: rows 64 MiB apart, the last one 4 GiB behind the first
    step = x[M - 1 - (64 << 16)::1 << 16]
    got = lin(step, dtype=F32)
    _check_product(got[-1:], tail[-1:].to(F64), w64)
    assert not got[:-1].any()
    assert torch.equal(mx4.quantise(step).codes[-1], q.codes[-1])


def test_weights_past_4_gib(gpu_device):
    """Packed weights whose last tiles lie past 2^32 bytes, few rows and many."""
    N, K = (1 << 21) + (1 << 14) + 5, 4096
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=gpu_device)
    scales = torch.full((N, K // 32), 120, dtype=torch.uint8, device=gpu_device)
    last = _weights(40, K, 42)
    codes[-40:], scales[-40:] = last.codes.to(gpu_device), last.scales.to(gpu_device)
    lin = mx4.Linear(mx4.Mx4(codes, scales))
    del codes, scales
    w64 = R.values(last.codes, last.scales).to(F64)
    for rows in (1, 20, 70):
        x = torch.randn(rows, K, generator=_gen(43)).to(BF)
        got = lin(x.to(gpu_device), dtype=F32)
        _check_product(got[:, -40:], x.to(F64), w64)
        assert not got[:, :-40].any()


def test_experts_of_the_most_rows(gpu_device):
    """65,535 rows, whose f32 outputs before the mix pass 4 GiB."""
    rows, E, k, H, I = 65535, 3, 4, 4096, 32
    ex, values = _experts(E, H, I, 44, gpu_device)
    x = torch.randn(rows, H, generator=_gen(45)).to(BF).to(gpu_device)
    ids, weights = _choice(rows, E, k, 46, gpu_device, repeat=True)
    got = ex(x, ids, weights)
    for part in (slice(0, 50), slice(rows - 50, rows)):
        _check_experts(got[part], x[part], ids[part], weights[part], values)


@pytest.mark.parametrize("rows", [4, 60, 300])
def test_experts_strided_rows(gpu_device, rows):
    """Rows, ids and weights taken out of wider tensors, reversed or every second one."""
    E, k, H, I = 7, 3, 96, 64
    ex, values = _experts(E, H, I, 47, gpu_device)
    wide = torch.randn(rows, H + 40, generator=_gen(48)).to(BF).to(gpu_device)
    ids, weights = _choice(2 * rows, E, k, 49, gpu_device)
    for x in (wide[:, 8:8 + H], wide[:, 3:3 + H], wide.flip(0)[:, :H], wide[:1, :H].expand(rows, H)):
        _check_experts(ex(x, ids[::2], weights[::2]), x.contiguous(), ids[::2], weights[::2], values)


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,K,N", [(2050, 96, 4100), (4001, 160, 8512), (1900, 544, 4500),
                                   (2048, 128, 4097)])
def test_linear_last_blocks(gpu_device, M, K, N, both):
    """Products of a few blocks more than the compute units hold at a time, whose last
    blocks run in parts: every row and column, with rows and columns that end in each part."""
    g = torch.Generator(device=gpu_device).manual_seed(M)
    w = mx4.quantise(torch.randn(N, K, generator=g, device=gpu_device) * 0.05)
    x = torch.randn(M, K, generator=g, device=gpu_device).to(BF)
    x64 = x.double()
    if both:
        x = mx4.quantise(x)
        x64 = x.dequantise().double()
    wt = w.dequantise().double().t().contiguous()
    want, size = x64 @ wt, x64.abs() @ wt.abs()
    for dtype in (F32, BF):
        got = mx4.Linear(w)(x, dtype=dtype).double()
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2 * K * 2.0 ** -24 * size
        assert ((got - want).abs() <= bound * 1.01).all()


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 2048, 40), (7, 2080, 1000), (16, 2272, 4096), (17, 2048, 33),
                                   (32, 4128, 2048), (33, 2048, 1360), (33, 2048, 1370),
                                   (64, 2176, 500)])
def test_linear_of_few_long_rows(gpu_device, M, K, N, both):
    """Few rows and columns of a long K: a block of eight waves each, rows in sixteens."""
    w = _weights(N, K, M + N)
    x = torch.randn(M, K, generator=_gen(K + M)).to(BF)
    x64 = x.to(F64)
    x = x.to(gpu_device)
    if both:
        x = mx4.quantise(x)
        x64 = x.dequantise().cpu().to(F64)
    lin = mx4.Linear(_to(w, gpu_device))
    for dtype in (BF, F32):
        _check_product(lin(x, dtype=dtype), x64, R.values(w.codes, w.scales).to(F64))


# -------------------------------------------------------------- other streams
def _busy(dev):
    """Work of some 100 ms on the current stream."""
    a = torch.ones(8192, 8192, device=dev)
    for _ in range(16):
        torch.mm(a, a)


def test_experts_errors_of_another_stream(gpu_device):
    """check_errors waits for calls of every stream, not for the current one's alone."""
    ex, _ = _experts(4, 64, 32, 60, gpu_device)
    x = torch.randn(5, 64, generator=_gen(61)).to(BF).to(gpu_device)
    ids, weights = _choice(5, 4, 3, 62, gpu_device)
    ids[2, 1] = 4
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy(gpu_device)
        y = ex(x, ids, weights)
    with pytest.raises(RuntimeError, match="id outside"):
        ex.check_errors()
    assert side.query()
    ex.check_errors()
    assert y.isfinite().all()


def test_handles_made_on_another_stream(gpu_device):
    """A handle's weights are laid out once it is there, whichever stream calls it first."""
    parts = [mx4.quantise((torch.randn(6, *s, generator=_gen(63)) * 0.1).to(gpu_device))
             for s in [(96, 256), (96, 256), (256, 96)]]
    w = mx4.quantise((torch.randn(700, 256, generator=_gen(64)) * 0.1).to(gpu_device))
    x = torch.randn(40, 256, generator=_gen(65)).to(BF).to(gpu_device)
    ids, weights = _choice(40, 6, 3, 66, gpu_device)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for make, args in ((lambda: mx4.Linear(w), (x,)),
                       (lambda: mx4.Experts(*parts), (x, ids, weights))):
        with torch.cuda.stream(side):
            _busy(gpu_device)
            handle = make()
        got.append(handle(*args))
        torch.cuda.synchronize()
        assert torch.equal(got[-1], handle(*args))
    _check_experts(got[1], x, ids, weights, [p.dequantise().double() for p in parts])
    _check_product(got[0], x.cpu().to(F64), w.dequantise().double().cpu())


# --------------------------------------- forms that few of the sizes above choose
def _form(M, K, N, both):
    """Rows and columns of a block, parts of K, blocks that run in quarters."""
    import ctypes

    from tilefoundry_amd._lib import lib

    form = (ctypes.c_int32 * 4)()
    lib().tfd_mx4_gemm_form(int(both), M, K, N, form)
    return list(form)


def _tile_rows(rows, E, k, H, I):
    from tilefoundry_amd._lib import lib

    return lib().tfd_mx4_experts_tile_rows(rows, k, E, H, I)


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,K,N", [(1270, 544, 8500), (1200, 288, 8300), (1152, 96, 9600),
                                   (1153, 1312, 8449)])
def test_linear_of_192_columns(gpu_device, M, K, N, both):
    """Blocks of 128 x 192: the last column block part full, rows that end inside a tile, K that
    is no multiple of a block; every output."""
    assert _form(M, K, N, both) == [128, 192, 1, 0]
    g = torch.Generator(device=gpu_device).manual_seed(M)
    w = mx4.quantise(torch.randn(N, K, generator=g, device=gpu_device) * 0.05)
    x = torch.randn(M, K, generator=g, device=gpu_device).to(BF)
    x64 = x.double()
    if both:
        x = mx4.quantise(x)
        x64 = x.dequantise().double()
    wt = w.dequantise().double().t().contiguous()
    want, size = x64 @ wt, x64.abs() @ wt.abs()
    lin = mx4.Linear(w)
    for dtype in (F32, BF):
        got = lin(x, dtype=dtype)
        bound = torch.finfo(dtype).eps / 2 * want.abs() + 2 * K * 2.0 ** -24 * size
        assert ((got.double() - want).abs() <= bound * 1.01).all()
        assert torch.equal(got, lin(x, dtype=dtype))


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("M,K,N", [(66, 2176, 70), (128, 6144, 260), (300, 4128, 513)])
def test_linear_in_parts(gpu_device, M, K, N, both):
    """Products that do split K, with their work and without."""
    import ctypes

    from tilefoundry_amd import _lib
    from tilefoundry_amd._lib import lib, ptr

    assert _form(M, K, N, both)[2] > 1
    w = mx4.quantise((torch.randn(N, K, generator=_gen(K)) * 0.05).to(gpu_device))
    x = torch.randn(M, K, generator=_gen(M)).to(BF).to(gpu_device)
    given = mx4.quantise(x) if both else x
    x64 = (given.dequantise() if both else x).double().cpu()
    w64 = w.dequantise().double().cpu()
    lin = mx4.Linear(w)
    need = lib().tfd_mx4_gemm_work_bytes(M, K, N)
    rows, scales = (given.codes, given.scales) if both else (x, None)
    for size in (need, 0):
        work = torch.full((need + 64,), 255, dtype=torch.uint8, device=gpu_device)
        out = torch.full((M + 1, N + 3), 7.0, device=gpu_device)
        a = _lib.TfdMx4GemmArgs(ptr(rows), rows.shape[1], ptr(scales), K // 32 if both else 0,
                                ptr(lin.packed), M, K, N, ptr(out), N + 3, _lib.TYPE_F32,
                                ptr(work) if size else None, size)
        lib().tfd_mx4_gemm(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
        _check_product(out[:M, :N], x64, w64)
        assert (out[M:] == 7).all() and (out[:, N:] == 7).all()
        assert (work[need:] == 255).all()
        if size:
            assert torch.equal(lin(given, dtype=F32), out[:M, :N])


# lists in tiles of 16: many experts, few rows each; H and I end inside a block of 128
LISTS = [(40, 64, 4, 1056, 96), (64, 72, 10, 4096, 160), (100, 300, 3, 416, 32)]


def _crowded(ids):
    """Some experts with more rows than a tile of 16: the first place of 17 rows, the second
    of 33."""
    ids = ids.clone()
    ids[:17, 0], ids[:33, 1] = 3, 5
    return ids


@pytest.mark.parametrize("rows,E,k,H,I", LISTS)
def test_experts_in_lists_of_16(gpu_device, rows, E, k, H, I):
    assert _tile_rows(rows, E, k, H, I) == 16
    ex, values = _experts(E, H, I, 70, gpu_device)
    x = torch.randn(rows, H, generator=_gen(71)).to(BF).to(gpu_device)
    ids, weights = _choice(rows, E, k, 72, gpu_device)
    ids = _crowded(ids)
    for dtype in (BF, F32):
        got = ex(x, ids, weights, dtype=dtype)
        _check_experts(got, x, ids, weights, values)
        assert torch.equal(got, ex(x, ids, weights, dtype=dtype))
    # against the definition, row by row, of which _check_experts is another writing.  `size` is
    # the sum with every magnitude in it: as t <= 2 silu(t) for t >= 0, |h| is at most twice its
    # hidden value.  Both sides round h to bf16, next to a border to either side: 2 * 2^-8 of h.
    # Sums' roundings: 2 H 2^-24 of the magnitudes in a (slope of the SiLU up to 1.1) and in b,
    # 2 I 2^-24 of those in y, under 8 (H + I) 2^-24 of 2 size together
    pick = torch.tensor([0, 16, 32, rows - 1], device=gpu_device)
    got = ex(x, ids, weights, dtype=F32)[pick].cpu().double()
    v = [t.cpu() for t in values]
    want = R.experts(x[pick], ids[pick], weights[pick], *v)
    size = R.experts(x[pick].abs(), ids[pick], weights[pick].abs(), *[t.abs() for t in v],
                     hidden_dtype=None)
    assert ((got - want).abs() <= 2 * size * (2.0 ** -7 + 8 * (H + I) * 2.0 ** -24)).all()
    # empty places, rows of nothing else, an expert several times in a row, one for all rows
    for seed, empty, repeat in [(1, 0.4, False), (2, 0.0, True), (3, 0.7, True)]:
        ids, weights = _choice(rows, E, k, seed, gpu_device, empty, repeat)
        ids[rows // 2] = -1
        got = ex(x, ids, weights)
        _check_experts(got, x, ids, weights, values)
        assert (got[rows // 2] == 0).all()
    for only in (0, E - 1):
        ids.fill_(only)
        _check_experts(ex(x, ids, weights), x, ids, weights, values)
    ids.fill_(-1)
    weights.fill_(math.nan)
    assert (ex(x, ids, weights) == 0).all()
    ex.check_errors()


@pytest.mark.parametrize("rows,E,k,H,I", LISTS)
def test_experts_in_lists_of_16_hard_rows(gpu_device, rows, E, k, H, I):
    """Ids outside the experts, values that are not finite, rows and places out of wider
    tensors, and the C entry that adds into padded rows."""
    import ctypes

    from tilefoundry_amd import _lib
    from tilefoundry_amd._lib import lib, ptr

    assert _tile_rows(rows, E, k, H, I) == 16
    ex, values = _experts(E, H, I, 73, gpu_device)
    base = torch.full((rows, H + 64), math.nan, dtype=BF)
    base[:, 16:16 + H] = torch.randn(rows, H, generator=_gen(74)).to(BF)
    base[0, 20], base[3, 30] = math.nan, math.inf
    x = base.to(gpu_device)[:, 16:16 + H]
    ids, weights = _choice(2 * rows, E, k, 75, gpu_device)
    ids, weights = ids[::2], weights[::2]
    crowd = _crowded(ids)
    got = ex(x, crowd, weights, dtype=F32)
    keep = torch.tensor([r for r in range(rows) if r not in (0, 3)], device=gpu_device)
    assert got[0].isnan().all() and not got[3].isfinite().any()
    _check_experts(got[keep], x[keep], crowd[keep], weights[keep], values)
    clean = x.clone()
    clean[0], clean[3] = clean[1], clean[2]
    for bad in (E, -2, 2 ** 31 - 1, -2 ** 31):
        wrong = crowd.clone()
        wrong[rows - 1, 1] = bad
        _check_experts(ex(clean, wrong, weights), clean, wrong, weights, values)
        with pytest.raises(RuntimeError, match="id outside"):
            ex.check_errors()
    wide_i = torch.full((rows, k + 2), 999, dtype=torch.int32, device=gpu_device)
    wide_w = torch.full((rows, k + 2), math.nan, device=gpu_device)
    wide_i[:, :k], wide_w[:, :k] = crowd, weights
    need = lib().tfd_mx4_experts_work_bytes(rows, k, E, H, I)
    work = torch.full((need + 256,), 255, dtype=torch.uint8, device=gpu_device)
    for dtype, kind in ((BF, _lib.TYPE_BF16), (F32, _lib.TYPE_F32)):
        for accumulate in (0, 1):
            out = torch.randn(rows + 2, H + 6, generator=_gen(76)).to(dtype).to(gpu_device)
            before = out.clone()
            a = _lib.TfdMx4ExpertsArgs(ptr(clean), H, ptr(wide_i), ptr(wide_w), k + 2,
                                       ptr(ex.w_gu), ptr(ex.w_down), rows, k, E, H, I, ptr(out),
                                       H + 6, kind, accumulate, 0.22, ptr(work), need, None)
            lib().tfd_mx4_experts(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
            _check_experts(out[:rows, :H], clean, crowd, weights, values, mult=0.22,
                           start=before[:rows, :H] if accumulate else None)
            assert torch.equal(out[rows:], before[rows:])
            assert torch.equal(out[:, H:], before[:, H:])
            assert (work[need:] == 255).all()


def test_experts_in_lists_of_16_replay(gpu_device):
    """The same bits from two streams at once and from two graphs that share the handle."""
    rows, E, k, H, I = LISTS[0]
    assert _tile_rows(rows, E, k, H, I) == 16
    ex, _ = _experts(E, H, I, 77, gpu_device)
    xs = torch.randn(4, rows, H, generator=_gen(78)).to(BF).to(gpu_device)
    picks = [_choice(rows, E, k, 79 + i, gpu_device) for i in range(4)]
    want = [ex(x, *p) for x, p in zip(xs, picks)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(ex(xs[i], *picks[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    graphs = []
    for _ in range(2):
        static = [xs[0].clone(), picks[0][0].clone(), picks[0][1].clone()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ex(*static)
        graphs.append((g, static, y))
    for i in (1, 2, 3):
        for g, static, y in graphs:
            for t, v in zip(static, (xs[i], *picks[i])):
                t.copy_(v)
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for _, _, y in graphs)


@pytest.mark.parametrize("tile,counts", [
    (64, [20, 40, 60, 70, 100, 0, 1]), (128, [129, 170, 200, 250, 20, 50, 300, 120, 0, 300])])
def test_experts_tiles_of_every_height(gpu_device, tile, counts):
    """Experts' rows that make tiles of each number of sixteens: up to 64 of 20 to 64 rows, up
    to 128 of 20, 49, 50 and 74 (five sixteens) to 128."""
    rows, E, k, H, I = sum(counts), len(counts), 1, 160, 96
    assert _tile_rows(rows, E, k, H, I) == tile
    ex, values = _experts(E, H, I, 80, gpu_device)
    x = torch.randn(rows, H, generator=_gen(81)).to(BF).to(gpu_device)
    ids = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    ids = ids[torch.randperm(rows, generator=_gen(82))].to(torch.int32).unsqueeze(1).to(gpu_device)
    weights = torch.randn(rows, k, generator=_gen(83)).to(gpu_device)
    for dtype in (BF, F32):
        _check_experts(ex(x, ids, weights, dtype=dtype), x, ids, weights, values)


@pytest.mark.parametrize("R,E,k,H,I", [(17, 8, 4, 64, 512), (11, 14, 12, 256, 1024),
                                       (90, 40, 3, 512, 64)])
def test_experts_workspace_serves_fewer_rows(gpu_device, R, E, k, H, I):
    """One workspace, of R rows: calls of any number up to that stay inside it."""
    import ctypes

    from tilefoundry_amd import _lib
    from tilefoundry_amd._lib import lib, ptr

    need = lib().tfd_mx4_experts_work_bytes(R, k, E, H, I)
    work = torch.full((need + 4096,), 165, dtype=torch.uint8, device=gpu_device)
    ex, values = _experts(E, H, I, 84, gpu_device)
    for rows in (R, R - 1, 16, 10, 1):
        if rows > R:
            continue
        x = torch.randn(rows, H, generator=_gen(85)).to(BF).to(gpu_device)
        ids, weights = _choice(rows, E, k, 86, gpu_device)
        out = torch.empty(rows, H, device=gpu_device)
        a = _lib.TfdMx4ExpertsArgs(ptr(x), H, ptr(ids), ptr(weights), k, ptr(ex.w_gu),
                                   ptr(ex.w_down), rows, k, E, H, I, ptr(out), H, _lib.TYPE_F32,
                                   0, 1.0, ptr(work), need, None)
        lib().tfd_mx4_experts(ctypes.addressof(a), torch.cuda.current_stream().cuda_stream)
        _check_experts(out, x, ids, weights, values)
        assert (work[need:] == 165).all()
