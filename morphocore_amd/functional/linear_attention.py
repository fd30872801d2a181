"""Linear attention with a decay for each head. No reference counterpart."""
from typing import Optional, Tuple, Union

import torch

from ._ops import ops


def linear_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, log_decay: torch.Tensor, state: Optional[torch.Tensor] = None,
                     offsets: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     final_state: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``S_t = exp(log_decay) S_(t-1) + k_t v_t^T``, ``out_t = scale q_t S_t`` for each head: every token attends to itself and
    those before it. Returns out, or (out, last state) with ``final_state``. Computed chunk by chunk with float32 sums and
    states; gradients flow to query, key, value and state, through out and the last state.

    query : [batch, tokens, heads, dim] float32, float16 or bfloat16 on a HIP device.
    key, value : [batch, tokens, kv_heads, dim], [batch, tokens, kv_heads, value_dim]; heads is a multiple of kv_heads, and
        neighbouring heads share keys and values. dim and value_dim up to 256.
    log_decay : [heads] float32, at most 0. No gradient.
    state : [batch, heads, dim, value_dim] float32 before the first token; zeros without it.
    offsets : [sequences + 1] int32 or int64 that do not fall, for sequences packed one after another: query, key and value are then
        [tokens, heads, dim] and sequence s is the rows from offsets[s] to offsets[s + 1] (it may have none); states are
        [sequences, ...]. Rows of no sequence get zeros.
    scale : 1 / sqrt(dim) by default.
    """
    out, last = ops.linear_attention(query, key, value, log_decay, state, offsets, scale, final_state)
    return (out, last) if final_state else out


def linear_attention_step(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor,
                          slots: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """One token of :func:`linear_attention` for each sequence of a batch: updates ``state`` in place and returns out
    [batch, heads, value_dim]. Not differentiable.

    query, key, value : [batch, heads, dim], [batch, kv_heads, dim], [batch, kv_heads, value_dim].
    state : [slots, heads, dim, value_dim] float32, each head's dense; no two of them may share memory.
    slots : [batch] int32 or int64, the sequences' places in ``state``; without it they are the batch's. A place outside it stands for
        no sequence (a padded batch) and gets zeros. Tokens that name the same place are taken one after another.
    """
    return ops.linear_attention_step(query, key, value, log_decay, state, slots, scale)
