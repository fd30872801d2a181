import torch
import torch.nn as nn

from ..functional import rms_norm


class RMSNorm(nn.Module):
    """Root-mean-square norm of the last dimension (:func:`morphocore_amd.functional.rms_norm`) with a
    learnable scale ``weight`` of shape (channels,), ones at first. ``forward(x, residual=None)`` returns y, or
    (y, x + residual) with a residual. No reference counterpart.
    """

    def __init__(self, channels: int, eps: float = 1e-6, dtype: torch.dtype = torch.float32):
        super().__init__()
        if channels < 1:
            raise ValueError(f"RMSNorm needs at least one channel, got {channels}")
        self.weight = nn.Parameter(torch.ones(channels, dtype=dtype))
        self.eps = eps

    def forward(self, x: torch.Tensor, residual: torch.Tensor = None):
        return rms_norm(x, self.weight, residual, self.eps)
