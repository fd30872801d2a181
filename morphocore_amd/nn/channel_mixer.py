import math

import torch
import torch.nn as nn

from ..functional import gated_silu8, linear8, rms_norm8
from .rms_norm import RMSNorm


class ChannelMixer(nn.Module):
    """Gated mixing of channels with a residual, the block between per-channel morphological layers; what it
    keeps for the backward of its four operators is in 8 bits, but for the residual sum itself:

        h = x + residual;  y = rms_norm(h);  z = gated_silu(y @ expand^T);  returns (z @ contract^T, h)

    so that the next block takes the two as its ``x`` and ``residual``. No reference counterpart.

    ``ChannelMixer(channels, hidden, eps=1e-6, dtype=torch.float32)``: parameters ``norm.weight`` (channels,),
    ``expand`` (2 hidden, channels), the gate's rows first, and ``contract`` (channels, hidden), the
    products' as uniform as nn.Linear's. Channels are the last dimension; with ``channels_first`` the input is
    [N, C, H, W] as the morphological layers', and moved to the end and back.
    """

    def __init__(self, channels: int, hidden: int, eps: float = 1e-6, dtype: torch.dtype = torch.float32, channels_first: bool = False):
        super().__init__()
        if channels < 1 or hidden < 1:
            raise ValueError(f"ChannelMixer needs at least one channel and one hidden channel, got {channels} and {hidden}")
        self.norm = RMSNorm(channels, eps, dtype)
        self.expand = nn.Parameter(torch.empty(2 * hidden, channels, dtype=dtype).uniform_(-1 / math.sqrt(channels), 1 / math.sqrt(channels)))
        self.contract = nn.Parameter(torch.empty(channels, hidden, dtype=dtype).uniform_(-1 / math.sqrt(hidden), 1 / math.sqrt(hidden)))
        self.channels_first = channels_first

    def forward(self, x: torch.Tensor, residual: torch.Tensor = None):
        if self.channels_first:
            x = x.movedim(1, -1)
            residual = residual.movedim(1, -1) if residual is not None else None
        y, packed, h = rms_norm8(x, self.norm.weight, residual, self.norm.eps)
        z, packed_z = gated_silu8(linear8(y, self.expand, packed))
        out = linear8(z, self.contract, packed_z)
        h = x if h is None else h
        if self.channels_first:
            out, h = out.movedim(-1, 1).contiguous(), h.movedim(-1, 1).contiguous()
        return out, h
