"""Microscaled 4-bit tensors (OCP MXFP4) on the GPU: quantisation and its inverse.

Along the last dimension 32 elements share a power-of-two scale (an e8m0 byte) and an
element is an e2m1 code, two to a byte: 17 bytes where bf16 takes 64.  ``quantise`` gives
codes and scales; ``Mx4.dequantise`` the values they stand for.  The kernels and their
exact definitions are declared in ``include/tf_mx4.h``.  ``Linear`` multiplies by mx4
weights, ``Experts`` runs a mixture's routed experts over them.

Every call runs on its tensors' device and that device's current stream, allocates its
outputs like any torch operation (so calls can be captured into a HIP graph and made from
several streams) and computes no gradients.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import lib, ptr

BLOCK = _lib.MX4_BLOCK
U8 = torch.uint8
TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16,
         torch.float16: _lib.TYPE_F16}


_current_device = torch.cuda.current_device
# the handle that torch.cuda.current_stream(device).cuda_stream gives, without the object
_raw_stream = torch._C._cuda_getCurrentRawStream


def launch(i: int, entry, *args) -> None:
    """Calls a C entry on the current stream of device *i*, with the device the current one
    (a launch belongs to the current device, a stream to its own)."""
    if i == _current_device():
        entry(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            entry(*args, _raw_stream(i))


def check_input(x, what: str, dtypes) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: expected a tensor, got {type(x).__name__}")
    if x.dtype not in dtypes:
        raise ValueError(f"{what}: dtype {x.dtype} is not one of "
                         f"{', '.join(str(d) for d in dtypes)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: these operators compute no gradients; detach it or work "
                         "under torch.no_grad()")
    # (a dual tensor keeps its tangent under no_grad too; without a level there is none)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"{what}: these operators compute no gradients; detach it")


def check_device(device, *others) -> None:
    if device.type != "cuda":
        raise ValueError(f"expected tensors on the GPU, got one on {device}")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and on {t.device}")


def check_apart(tensors, what: str) -> None:
    """Contiguous tensors that a call writes side by side share no memory."""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                   for t in tensors if t.numel())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"{what}: two of the tensors overlap in memory")


# what the C entries take as 32-bit integers (ctypes would cut a larger one to its low bits)
LONGEST = (1 << 31) - 1                      # values of a row
MAX_K, MAX_N = 1 << 22, 1 << 24              # of a product
MAX_EXPERT = 1 << 20                         # hidden columns, an expert's width


def check_row(K: int, what: str) -> None:
    if K > LONGEST:
        raise ValueError(f"{what}: the last dimension must be below 2^31, got {K}")


WIDEST = 1 << 23                             # elements between rows that a product takes


def rows_of(x: torch.Tensor, align: int = 1, widest: int = 1 << 62) -> torch.Tensor:
    """*x* as rows of its last dimension with unit stride, rows that do not overlap and,
    with *align*, that start at multiples of that many bytes: *x* itself where it is that
    (contiguous in any number of dimensions), else a two-dimensional view or, where its rows
    lie otherwise or more than *widest* elements apart, a copy."""
    if x.is_contiguous() and (align == 1 or not x.data_ptr() % align and (
            not x.shape[-1] * x.element_size() % align or x.numel() == x.shape[-1])):
        return x
    K = x.shape[-1]
    x = x.reshape(-1, K)
    size = x.element_size()
    if (x.stride(1) != 1 and K > 1) or (x.shape[0] > 1 and (
            not K <= x.stride(0) <= widest or x.stride(0) * size % align)) or x.data_ptr() % align:
        return x.clone(memory_format=torch.contiguous_format)
    return x


def row_stride(x: torch.Tensor) -> int:
    """Elements from one row of ``rows_of`` to the next."""
    return x.shape[-1] if x.is_contiguous() else x.stride(-2)


class Mx4:
    """Codes uint8 ``[..., K / 2]`` and scales uint8 ``[..., K / 32]`` of one tensor."""

    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        c, s = codes, scales
        if c.dtype != U8 or s.dtype != U8:
            raise ValueError(f"mx4 codes and scales are uint8, got {c.dtype} and {s.dtype}")
        if c.dim() < 1 or c.shape[:-1] != s.shape[:-1] or c.shape[-1] != 16 * s.shape[-1] or \
                c.shape[-1] == 0:
            raise ValueError(f"mx4 codes {tuple(c.shape)} and scales {tuple(s.shape)} are not "
                             "[..., K / 2] and [..., K / 32] of one tensor")
        if c.device != s.device:
            raise ValueError(f"mx4 codes on {c.device}, scales on {s.device}")
        self.codes, self.scales = c, s

    @classmethod
    def _of(cls, codes, scales) -> "Mx4":
        """Of tensors made for each other."""
        t = cls.__new__(cls)
        t.codes, t.scales = codes, scales
        return t

    def __repr__(self) -> str:
        return f"Mx4(shape={self.shape}, device={self.device})"

    @property
    def shape(self) -> tuple[int, ...]:
        """Shape of the values."""
        return (*self.codes.shape[:-1], 2 * self.codes.shape[-1])

    @property
    def device(self):
        return self.codes.device

    def __getitem__(self, index) -> "Mx4":
        """The tensors of some of the leading dimensions' entries."""
        if self.codes.dim() < 2:
            raise IndexError("mx4: an index takes whole rows, this is one row")
        return Mx4(self.codes[index], self.scales[index])

    def dequantise(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, exact in f32 and bf16 (f16 rounds what its range does not hold)."""
        if dtype not in TYPES:
            raise ValueError(f"dequantise: dtype {dtype} is not one of "
                             f"{', '.join(str(d) for d in TYPES)}")
        shape = self.shape
        check_row(shape[-1], "dequantise")
        codes, scales = rows_of(self.codes, 4), rows_of(self.scales)
        if not codes.is_cuda:
            check_device(codes.device)
        out = codes.new_empty(shape, dtype=dtype)
        K = shape[-1]
        launch(codes.get_device(), lib().tfd_mx4_dequantise, ptr(codes), row_stride(codes), ptr(scales),
               row_stride(scales), out.numel() // K, K, ptr(out), K, TYPES[dtype])
        return out


def quantise(x: torch.Tensor) -> Mx4:
    """Rows ``[..., K]`` (f32, bf16 or f16, K a multiple of 32) to mx4: for 32 values with
    largest magnitude t the scale 2^(floor(log2 t) - 2), codes rounded to nearest even,
    magnitudes past 6 scales as 6.  A block with a value that is not finite becomes NaN.
    Up to 2^35 - 2048 values a call, rows below 2^31."""
    check_input(x, "quantise", TYPES)
    *lead, K = x.shape if x.dim() else (0,)
    if K % BLOCK or K == 0:
        raise ValueError(f"quantise: the last dimension must be a multiple of {BLOCK}, got "
                         f"{tuple(x.shape)}")
    check_row(K, "quantise")
    if not x.is_cuda:
        check_device(x.device)
    codes = x.new_empty((*lead, K // 2), dtype=U8)
    scales = x.new_empty((*lead, K // BLOCK), dtype=U8)
    rows = rows_of(x)
    launch(x.get_device(), lib().tfd_mx4_quantise, ptr(rows), row_stride(rows), TYPES[x.dtype],
           x.numel() // K, K, ptr(codes), K // 2, ptr(scales), K // BLOCK)
    return Mx4._of(codes, scales)


def _pack(first: Mx4, second: Mx4 | None, what: str) -> torch.Tensor:
    """Weights ``[..., N, K]`` (two of them alternating row by row) in the products'
    layout, once, at load time."""
    check_device(first.device, *(() if second is None else (second.codes,)))
    K = first.shape[-1]
    parts = [t.contiguous() for w in (first, second) if w is not None
             for t in (w.codes, w.scales)]
    for i in (0, 2):
        if i < len(parts) and parts[i].data_ptr() % 16:
            parts[i] = parts[i].clone()
    rows = first.codes.numel() // (K // 2)
    if rows == 0:
        raise ValueError(f"{what}: no rows in weights of shape {first.shape}")
    L = lib()
    packed = torch.empty(L.tfd_mx4_packed_bytes(rows * (len(parts) // 2), K), dtype=U8,
                         device=first.device)
    parts += [None] * (4 - len(parts))
    launch(first.codes.get_device(), L.tfd_mx4_pack, *(ptr(t) for t in parts), rows, K, ptr(packed))
    return packed


def _settle(device) -> None:
    """Waits, at load time, for what the current stream makes of a handle: its first call may
    be on another one.  (A handle made inside a capture is that graph's.)"""
    with torch.cuda.device(device):
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().synchronize()


BF16, INT32, FLOAT32 = (torch.bfloat16,), (torch.int32,), (torch.float32,)
MAX_ROWS = 1 << 30
OUT_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16}


def _out_type(dtype, what: str) -> int:
    if dtype not in OUT_TYPES:
        raise ValueError(f"{what}: dtype {dtype} is neither float32 nor bfloat16")
    return OUT_TYPES[dtype]


class Linear:
    """x -> x W^T by mx4 weights ``[N, K]``, kept in the layout the kernels read.

    x: bf16 ``[..., K]`` (weights become bf16 on the way, exactly; an infinity where a scale byte
    past 252, which ``quantise`` never gives, takes one over its range), or an ``Mx4`` of that
    shape (both operands stay in 4 bits).  Sums are f32; the output is bf16 or f32."""

    def __init__(self, weight: Mx4):
        if len(weight.shape) != 2:
            raise ValueError(f"Linear: weights must be [N, K], got {weight.shape}")
        self.N, self.K = weight.shape
        if self.N > MAX_N or self.K > MAX_K:
            raise ValueError(f"Linear: weights of up to {MAX_N} x {MAX_K}, got {weight.shape}")
        self.device = weight.device
        self.packed = _pack(weight, None, "Linear")
        self.index = self.packed.get_device()
        _settle(self.device)

    def __call__(self, x, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        kind = _out_type(dtype, "Linear")
        scales, ldxs = None, 0
        if isinstance(x, Mx4):
            lead, K, values = x.shape[:-1], x.shape[-1], x.codes
        else:
            check_input(x, "Linear", BF16)
            if x.dim() < 1:
                raise ValueError("Linear: the input has no dimensions")
            lead, K, values = x.shape[:-1], x.shape[-1], x
        if K != self.K:
            raise ValueError(f"Linear: input {tuple(x.shape)} for weights [{self.N}, {self.K}]")
        if values.get_device() != self.index:
            raise ValueError(f"Linear: input on {values.device}, weights on {self.device}")
        values = rows_of(values, 16, WIDEST)
        if isinstance(x, Mx4):
            scales = rows_of(x.scales, 1, WIDEST)
            ldxs = row_stride(scales)
        out = values.new_empty((*lead, self.N), dtype=dtype)
        rows = out.numel() // self.N
        if rows > MAX_ROWS:
            raise ValueError(f"Linear: up to {MAX_ROWS} rows a call, got {rows}")
        L = lib()
        work, need = None, 0
        if rows > _lib.MX4_WHOLE_ROWS:
            need = L.tfd_mx4_gemm_work_bytes(rows, K, self.N)
            work = values.new_empty(need, dtype=U8) if need else None
        a = _lib.TfdMx4GemmArgs(ptr(values), row_stride(values), ptr(scales), ldxs,
                                ptr(self.packed), rows, K, self.N, ptr(out), self.N, kind,
                                ptr(work), need)
        launch(self.index, L.tfd_mx4_gemm, ctypes.addressof(a))
        return out


class Experts:
    """The routed experts of a mixture by mx4 weights: gate and up ``[E, I, H]``, down
    ``[E, H, I]``.  For each row of bf16 x ``[rows, H]``, with ids int32 and weights f32
    ``[rows, k]`` (``routing.Routing`` gives both),

        y = sum over the row's places of weight * down_e(silu(gate_e x) * (up_e x)).

    Sums are f32, the output rounded once to bf16 or f32.  The hidden values are the down
    product's operands: rounded to bf16, or in calls of up to 16 rows and 128 places kept as
    sums of two bf16 (2^-17); a row's last bits so depend on its call's rows.  Id -1 is an empty
    place; any other id outside the experts is skipped and makes ``check_errors`` raise.  An
    expert may come twice in a row.  A call takes up to 65,535 rows, whose x and hidden
    values are each below 2 GiB."""

    def __init__(self, gate: Mx4, up: Mx4, down: Mx4):
        if len(gate.shape) != 3 or gate.shape != up.shape or \
                down.shape != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise ValueError("Experts: gate and up must be [E, I, H] and down [E, H, I], got "
                             f"{gate.shape}, {up.shape}, {down.shape}")
        self.E, self.I, self.H = gate.shape
        if not 1 <= self.E <= _lib.ROUTE_MAX_EXPERTS:
            raise ValueError(f"Experts: 1 to {_lib.ROUTE_MAX_EXPERTS} experts, got {self.E}")
        if self.H > MAX_EXPERT or self.I > MAX_EXPERT:
            raise ValueError(f"Experts: hidden and width up to {MAX_EXPERT}, got {self.H} and "
                             f"{self.I}")
        check_device(gate.device, up.codes, down.codes)
        self.device = gate.device
        self.w_gu = _pack(gate, up, "Experts")
        self.w_down = _pack(down, None, "Experts")
        self.index = self.w_gu.get_device()
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        _settle(self.device)

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        kind = _out_type(dtype, "Experts")
        check_input(x, "x", BF16)
        check_input(ids, "ids", INT32)
        check_input(weights, "weights", FLOAT32)
        if x.dim() != 2 or x.shape[1] != self.H:
            raise ValueError(f"Experts: x must be [rows, {self.H}], got {tuple(x.shape)}")
        rows = x.shape[0]
        if ids.dim() != 2 or ids.shape != weights.shape or ids.shape[0] != rows or \
                not 1 <= ids.shape[1] <= 64:
            raise ValueError(f"Experts: ids {tuple(ids.shape)} and weights "
                             f"{tuple(weights.shape)} must be [{rows}, 1..64]")
        for t in (x, ids, weights):
            if t.get_device() != self.index:
                raise ValueError(f"Experts: input on {t.device}, weights on {self.device}")
        if rows > 65535:
            raise ValueError(f"Experts: up to 65535 rows a call, got {rows}")
        x = rows_of(x, 16, ((1 << 30) - 1) // max(rows, 1))
        ids, weights = ids.contiguous(), weights.contiguous()
        k, L = ids.shape[1], lib()
        out = x.new_empty((rows, self.H), dtype=dtype)
        need = L.tfd_mx4_experts_work_bytes(rows, k, self.E, self.H, self.I)
        # of the stream that uses it, like the output: calls on several streams and captured
        # graphs share nothing
        work = x.new_empty(need, dtype=U8)
        a = _lib.TfdMx4ExpertsArgs(
            ptr(x), row_stride(x), ptr(ids), ptr(weights), k, ptr(self.w_gu), ptr(self.w_down),
            rows, k, self.E, self.H, self.I, ptr(out), self.H, kind, 0, 1.0, ptr(work), need,
            ptr(self.err))
        launch(self.index, L.tfd_mx4_experts, ctypes.addressof(a))
        return out

    def check_errors(self) -> None:
        """Raises if a call since the last check met an id outside the experts (waits for
        the device: calls may be on any stream)."""
        torch.cuda.synchronize(self.device)
        if int(self.err.item()):
            self.err.zero_()
            torch.cuda.synchronize(self.device)      # before a call on another stream
            raise RuntimeError("mx4 experts: an id outside the experts (and not -1) was skipped")
