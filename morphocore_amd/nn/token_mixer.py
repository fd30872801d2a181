import math
from typing import Optional

import torch
import torch.nn as nn

from ..functional import (grid_positions, linear8, linear_attention, linear_attention_step, rms_norm, rms_norm8, rms_norm_rotary,
                          rotary_frequencies)
from .rms_norm import RMSNorm


class TokenMixer(nn.Module):
    """Mixing of tokens with a residual, beside :class:`ChannelMixer`, which mixes their channels; the projections keep their inputs in
    8 bits for the backward:

        h = x + residual;  y = rms_norm(h);  q, k, v = heads of y @ project^T;  q, k = rms_norm_rotary(q, k, positions)
        returns (linear_attention(q, k, v) @ contract^T, h)

    so that the next block takes the two as its ``x`` and ``residual``. A token attends to itself and to those before it, in the order
    of memory (of an image: rows, then columns). No reference counterpart.

    ``TokenMixer(channels, heads, axes=1, kv_heads=heads, dim=channels // heads, base=10000, eps=1e-6, dtype=torch.float32)``:
    parameters ``norm.weight`` (channels,), ``query_weight`` and ``key_weight`` (dim,), ``project`` ((heads + 2 kv_heads) dim, channels),
    the queries' rows first, then the keys', and ``contract`` (channels, heads dim), the products' as uniform as nn.Linear's; buffers
    ``log_decay`` (heads,) float32, whose heads remember 16 to 4096 tokens, and ``frequencies`` (axes, dim // 2) float64, the pairs
    shared out among the axes, the first ones' first. The buffers keep their types where the module's is changed.

    ``forward(x, residual=None, positions=None, state=None, offsets=None, final_state=False)``: x is [batch, places of each axis ...,
    channels], with ``channels_first`` [batch, channels, places of each axis ...], and ``positions`` the places by default, otherwise
    [places of each axis ..., axes] or [places, axes] with all of them in one dimension, either with the batch in front; with
    ``offsets`` it is [tokens, channels], sequences one after another, with their ``positions`` [tokens, axes]. Returns (out, h), with
    ``final_state`` (out, h, last states), which ``state`` of a later call goes on from.

    ``step(x, state, positions, residual=None, slots=None)``: a token of each sequence, x [batch, channels] and positions [batch, axes],
    without gradients; updates ``state`` [slots, heads, dim, dim] in place and returns (out, h).
    """

    def __init__(self, channels: int, heads: int, axes: int = 1, kv_heads: Optional[int] = None, dim: Optional[int] = None, base: float = 10000.0,
                 eps: float = 1e-6, dtype: torch.dtype = torch.float32, channels_first: bool = False):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channels < 1 or heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"TokenMixer needs channels and heads that are a multiple of kv_heads, got {channels}, {heads} and {kv_heads}")
        dim = channels // heads if dim is None else dim
        if axes < 1 or axes > 8 or dim // 2 < axes or dim > 256:
            raise ValueError(f"TokenMixer needs 1 to 8 axes, a pair of a head's values for each, and at most 256 values, got {axes} and {dim}")
        self.heads, self.kv_heads, self.dim, self.axes, self.channels_first = heads, kv_heads, dim, axes, channels_first
        self.norm = RMSNorm(channels, eps, dtype)
        self.query_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        self.key_weight = nn.Parameter(torch.ones(dim, dtype=dtype))
        rows, inner = (heads + 2 * kv_heads) * dim, heads * dim
        self.project = nn.Parameter(torch.empty(rows, channels, dtype=dtype).uniform_(-1 / math.sqrt(channels), 1 / math.sqrt(channels)))
        self.contract = nn.Parameter(torch.empty(channels, inner, dtype=dtype).uniform_(-1 / math.sqrt(inner), 1 / math.sqrt(inner)))
        each, more = divmod(dim // 2, axes)
        self.register_buffer("log_decay", -torch.exp2(-4 - 8 * torch.arange(heads, dtype=torch.float32) / max(heads - 1, 1)))
        self.register_buffer("frequencies", rotary_frequencies([each + (a < more) for a in range(axes)], base), persistent=False)

    def _apply(self, fn, recurse=True):
        kept = {name: getattr(self, name) for name in ("log_decay", "frequencies")}
        super()._apply(fn, recurse)
        for name, value in kept.items():
            moved = getattr(self, name)
            setattr(self, name, moved if moved.dtype == value.dtype else value.to(moved.device))
        return self

    def _normed(self, x: torch.Tensor, residual: Optional[torch.Tensor]):
        """The norm, its 8-bit form where a backward may read it, and the sum with the residual."""
        if torch.is_grad_enabled():
            y, packed, h = rms_norm8(x, self.norm.weight, residual, self.norm.eps)
            return y, packed, x if h is None else h
        y = rms_norm(x, self.norm.weight, residual, self.norm.eps)
        return (y, None, x) if residual is None else (y[0], None, y[1])

    def _rotated(self, y: torch.Tensor, packed, positions: torch.Tensor):
        qkv = linear8(y, self.project, packed).unflatten(-1, (self.heads + 2 * self.kv_heads, self.dim))
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), -2)
        return *rms_norm_rotary(q, k, self.query_weight, self.key_weight, positions, self.frequencies, self.norm.eps), v

    def forward(self, x: torch.Tensor, residual: torch.Tensor = None, positions: torch.Tensor = None, state: torch.Tensor = None,
                offsets: torch.Tensor = None, final_state: bool = False):
        if x.dim() != (2 if offsets is not None else 2 + self.axes):
            raise ValueError(f"TokenMixer expects {'[tokens, channels]' if offsets is not None else f'a batch with {self.axes} axes of places'}, got {list(x.shape)}")
        if offsets is not None and (positions is None or self.channels_first):
            raise ValueError("TokenMixer needs the positions of packed sequences, and their channels last")
        if self.channels_first:
            x = x.movedim(1, -1)
            residual = residual.movedim(1, -1) if residual is not None else None
        places = x.shape[1:-1]
        y, packed, h = self._normed(x, residual)
        if positions is None:
            positions = grid_positions(places, x.device)
        elif offsets is None and positions.shape[-1 - self.axes:-1] == places:
            positions = positions.flatten(-1 - self.axes, -2)
        if offsets is None:  # places of all axes become one dimension
            y, packed = y.flatten(1, -2), type(packed)(*(t.flatten(1, -2) for t in packed)) if packed is not None else None
        q, k, v = self._rotated(y, packed, positions)
        out = linear_attention(q, k, v, self.log_decay, state, offsets, final_state=final_state)
        out, last = out if final_state else (out, None)
        out = linear8(out.flatten(-2), self.contract)
        if offsets is None:
            out = out.unflatten(1, places)
        if self.channels_first:
            out, h = out.movedim(-1, 1).contiguous(), h.movedim(-1, 1).contiguous()
        return (out, h, last) if final_state else (out, h)

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: torch.Tensor, positions: torch.Tensor, residual: torch.Tensor = None, slots: torch.Tensor = None):
        if x.dim() != 2:
            raise ValueError(f"TokenMixer.step expects [batch, channels], got {list(x.shape)}")
        y, _, h = self._normed(x, residual)
        q, k, v = self._rotated(y, None, positions)
        out = linear_attention_step(q, k, v, self.log_decay, state, slots)
        return linear8(out.flatten(-2), self.contract), h
