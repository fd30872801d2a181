"""Root-mean-square norm of the last dimension. No reference counterpart."""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._ops import ops
from .checkpoint8 import Packed8


class Normed8(NamedTuple):
    """What :func:`rms_norm8` returns: ``y`` (None with ``full=False``), ``packed`` (y in 8-bit blocks) and
    the sum ``h`` (None without a residual)."""
    y: Optional[torch.Tensor]
    packed: Packed8
    h: Optional[torch.Tensor]


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, h = x + residual; returns y, or
    (y, h) with a residual. One pass over the data forward and one backward, sums in float64 forward (y is rounded
    once) and in float32 backward.

    x : [..., C] float32, float16 or bfloat16 on a HIP device.
    weight : [C], of x's type or float32.
    residual : of x's shape and type. h is returned in x's type (y is the norm of the unrounded sum).
    """
    y, h = ops.rms_norm(x, weight, residual, eps)
    return y if residual is None else (y, h)


def rms_norm8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
              full: bool = True) -> Normed8:
    """:func:`rms_norm` that also gives y in 8-bit blocks, from the same pass: the packed input of a
    :func:`linear8` that follows (y itself need not outlive it), or, with ``full=False`` and without
    gradients, the only output beside h. Gradients flow through y and h; ``packed`` has none.
    """
    y, h, codes, scales = ops.rms_norm8(x, weight, residual, eps, full)
    return Normed8(y, Packed8(codes, scales), h)
