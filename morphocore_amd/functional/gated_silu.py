"""The gated activation of a channel-mixing block. No reference counterpart."""
from typing import NamedTuple, Optional

import torch

from ._ops import ops
from .checkpoint8 import Packed8


class Gated8(NamedTuple):
    """What :func:`gated_silu8` returns: ``y`` and ``packed``, y in 8-bit blocks."""
    y: torch.Tensor
    packed: Packed8


def gated_silu(gate: torch.Tensor, up: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``gate * sigmoid(gate) * up``, computed in float32; without ``up``, ``gate`` holds both, [..., 2 C]: the
    gate in the first half of the last dimension. Slices of wider rows are read where they are.
    """
    return ops.gated_silu(gate, up)


def gated_silu8(gate: torch.Tensor, up: Optional[torch.Tensor] = None) -> Gated8:
    """:func:`gated_silu` that keeps gate and up in 8-bit blocks for its backward (2 bytes a pair instead of 4
    or 8) and also gives y in 8-bit blocks, the packed input of a :func:`linear8` that follows. The
    gradients are the activation's at the kept values; ``packed`` has none.
    """
    y, codes, scales = ops.gated_silu8(gate, up)
    return Gated8(y, Packed8(codes, scales))
