"""A linear layer that keeps its input in 8 bits. No reference counterpart."""
from typing import Optional

import torch

from ._ops import ops
from .checkpoint8 import Packed8


def grad_weight8(grad_output: torch.Tensor, packed: Packed8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The weight gradient of a linear layer, ``grad_output^T @ unpack8(packed)`` summed over all leading
    dimensions: [N, K] from grad_output [..., N] and a packed input [..., K]. Products are exact (float32
    gradients to 2^-133) and sums float32, rounded once to ``dtype``: grad_output's type (the default) or
    float32. Not differentiable.
    """
    return ops.grad_weight8(grad_output, packed.codes, packed.scales, dtype)


def linear8(x: torch.Tensor, weight: torch.Tensor, packed: Optional[Packed8] = None) -> torch.Tensor:
    """``x @ weight^T`` whose backward takes the weight's gradient from x in 8-bit blocks, all that is kept of it.

    x : [..., K] float32, float16 or bfloat16 on a HIP device. weight : [N, K] of the same type.
    The products, forward and backward, are the operands' type's, under autocast too.
    packed : x in 8-bit blocks where the operator before has made them (rms_norm8, gated_silu8); packed here otherwise.
    """
    codes, scales = packed if packed is not None else (None, None)
    return ops.linear8(x, weight, codes, scales)
