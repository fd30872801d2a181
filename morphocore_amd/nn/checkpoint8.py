import torch
import torch.nn as nn

from ..functional import checkpoint8


class Checkpoint8(nn.Module):
    """A module of one tensor to one tensor (a MorphoStack, an Opening, a Sequential of them) that keeps only
    its input, in 8 bits, and runs again in the backward (:func:`morphocore_amd.functional.checkpoint8`, which says
    what ``preserve_rng`` is).
    No reference counterpart."""

    def __init__(self, module: nn.Module, preserve_rng: bool = True):
        super().__init__()
        if not isinstance(module, nn.Module):
            raise TypeError(f"Checkpoint8 takes a module, not {type(module).__name__}")
        self.module = module
        self.preserve_rng = preserve_rng

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return checkpoint8(self.module, x, self.preserve_rng)
