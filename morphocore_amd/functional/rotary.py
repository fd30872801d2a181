"""Rotary positions with several axes, alone or with the norm of queries and keys. No reference counterpart."""
from typing import Sequence, Tuple

import torch

from ._ops import ops


def rotary_frequencies(pairs: Sequence[int], base: float = 10000.0, shared: bool = False, device=None) -> torch.Tensor:
    """The radians a position that :func:`axial_rotary` turns each pair of values by, [axes, sum(pairs)] float64:
    ``pairs[a]`` pairs of axis a (time, height, width, ...), one axis after another. Each axis goes from 1 down to
    ``base^-(1 - 1 / pairs[a])`` by itself; with ``shared`` the axes are sections of one such range over all pairs.
    """
    if not pairs or any(n < 0 for n in pairs):
        raise ValueError(f"rotary_frequencies needs a non negative number of pairs for each axis, got {list(pairs)}")
    total = sum(pairs)
    table = torch.zeros(len(pairs), total, dtype=torch.float64)
    first = 0
    for axis, n in enumerate(pairs):
        step = torch.arange(n, dtype=torch.float64)
        table[axis, first:first + n] = base ** (-(first + step) / total if shared else -step / max(n, 1))
        first += n
    return table.to(device)


def grid_positions(sizes: Sequence[int], device=None) -> torch.Tensor:
    """The positions of a grid's places (frames, rows, columns, ...), the last axis fastest: [product of sizes, axes] int32."""
    if not sizes:
        raise ValueError("grid_positions needs at least one axis")
    axes = torch.meshgrid(*(torch.arange(n, dtype=torch.int32, device=device) for n in sizes), indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], -1)


def axial_rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """Turns pair j of every head's values, (a, b), to (a cos - b sin, b cos + a sin) by the token's angle, the sum over the axes of
    ``positions[token, axis] * frequencies[axis, j]``. Angles are formed in float64, so positions may be far.

    x : [..., heads, values] float32, float16 or bfloat16 on a HIP device, up to 512 values.
    positions : [..., axes] int32, int64 or float32, of x's tokens (its dimensions before the heads) or of the last of them; up
        to 8 axes.
    frequencies : [axes, pairs] float64 (:func:`rotary_frequencies`). Values behind the pairs stay as they are.
    interleaved : pair j is values 2 j and 2 j + 1; otherwise j and pairs + j.
    """
    return ops.axial_rotary(x, positions, frequencies, interleaved)


def rms_norm_rotary(query: torch.Tensor, key: torch.Tensor, query_weight: torch.Tensor, key_weight: torch.Tensor, positions: torch.Tensor,
                    frequencies: torch.Tensor, eps: float = 1e-6, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`axial_rotary` of ``x / sqrt(mean(x^2) + eps) * weight`` over each head's values, of queries and keys in one pass;
    returns both. Nothing but the inputs is kept for the backward.

    query, key : [..., heads, values] with the same tokens and values and any numbers of heads; slices of one projection are
        read where they are.
    query_weight, key_weight : [values], of the queries' type or float32.
    """
    return ops.rms_norm_rotary(query, key, query_weight, key_weight, positions, frequencies, eps, interleaved)
