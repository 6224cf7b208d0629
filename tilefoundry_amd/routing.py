"""The choice of experts from a router's logits, on the device.

``Routing`` holds a model's rule -- how logits become scores, groups of experts, how many
are picked, what their weights are -- and is called with the logits (and a bias that
balances the choice without entering the weights).  The rule is ``tfd_route_experts``
(include/tf_mx4.h); the fixed routers of the two hybrid models stay ``tfd_route_topk``.

    routing = Routing(top_k=8, score="sigmoid", groups=8, kept_groups=4, scale=2.5)
    weights, ids = routing(logits, bias)         # f32 and int32, [rows, top_k + shared]

Places for which a mask left no expert hold id -1 and weight 0, which ``mx4.Experts`` skips.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import lib, ptr
from .mx4 import FLOAT32, TYPES, check_device, check_input, launch, row_stride, rows_of

MAX_ROWS = 4 * ((1 << 24) - 1)          # blocks of four rows, 32 bits of threads in a launch
SCORES = {"softmax": _lib.SCORE_SOFTMAX, "sigmoid": _lib.SCORE_SIGMOID}


@dataclass(frozen=True)
class Routing:
    """A routing rule; see the module docstring.

    ``score``: "softmax" over the row or "sigmoid" of each logit.  With ``groups`` > 1 the
    experts lie in that many equal runs; runs rank by the sum of their best ``group_top``
    choices and the best ``kept_groups`` stay.  ``renormalise`` divides the picks' scores by
    their sum; ``scale`` multiplies the weights.  ``shared`` experts follow the routed ones
    in every row, with weight 1.
    """

    top_k: int
    score: str = "softmax"
    groups: int = 1
    kept_groups: int = 1
    group_top: int = 2
    renormalise: bool = True
    scale: float = 1.0
    shared: int = 0

    def __post_init__(self):
        if self.score not in SCORES:
            raise ValueError(f"score must be one of {', '.join(SCORES)}, got {self.score!r}")
        if self.top_k < 1 or self.shared < 0 or self.top_k + self.shared > 64:
            raise ValueError(f"top_k {self.top_k} and shared {self.shared}: 1 to 64 places in "
                             "all, one routed at least")
        if not 1 <= self.groups <= 64 or not 1 <= self.kept_groups <= self.groups:
            raise ValueError(f"kept_groups must lie in 1..groups and groups in 1..64, got "
                             f"{self.kept_groups} of {self.groups}")
        if self.group_top not in (1, 2):
            raise ValueError(f"group_top must be 1 or 2, got {self.group_top}")
        if not 0 < self.scale < math.inf:
            raise ValueError(f"scale must be positive and finite, got {self.scale}")

    def __call__(self, logits: torch.Tensor, bias: torch.Tensor | None = None):
        """Logits ``[rows, experts]`` (f32, bf16 or f16) and the choice's bias f32
        ``[experts]`` -> weights f32 and ids int32, ``[rows, top_k + shared]``."""
        check_input(logits, "logits", TYPES)
        if logits.dim() != 2:
            raise ValueError(f"logits must be [rows, experts], got {tuple(logits.shape)}")
        rows, experts = logits.shape
        if rows > MAX_ROWS:
            raise ValueError(f"routing: up to {MAX_ROWS} rows a call, got {rows}")
        if not 1 <= experts <= _lib.ROUTE_MAX_EXPERTS or experts % self.groups:
            raise ValueError(f"{experts} experts: 1 to {_lib.ROUTE_MAX_EXPERTS}, a multiple of "
                             f"{self.groups} groups")
        if self.top_k > self.kept_groups * (experts // self.groups):
            raise ValueError(f"top_k {self.top_k} of {self.kept_groups} groups of "
                             f"{experts // self.groups} experts")
        if bias is not None:
            check_input(bias, "bias", FLOAT32)
            if bias.shape != (experts,):
                raise ValueError(f"bias must be [{experts}], got {tuple(bias.shape)}")
            bias = bias.contiguous()
            check_device(logits.device, bias)
        elif not logits.is_cuda:
            check_device(logits.device)
        logits = rows_of(logits)
        n = self.top_k + self.shared
        weights = logits.new_empty((rows, n), dtype=torch.float32)
        ids = logits.new_empty((rows, n), dtype=torch.int32)
        a = _lib.TfdRouteArgs(
            ptr(logits), row_stride(logits), TYPES[logits.dtype], ptr(bias), rows, experts,
            self.top_k, SCORES[self.score], self.groups, self.kept_groups, self.group_top,
            self.shared, int(self.renormalise), self.scale, ptr(weights), ptr(ids), n)
        launch(logits.get_device(), lib().tfd_route_experts, ctypes.addressof(a))
        return weights, ids
