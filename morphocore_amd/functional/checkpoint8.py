"""Activations kept in 8 bits: the blocks themselves, and a layer whose input is all that it keeps.

No reference counterpart: its layers keep their inputs and outputs as they are for the backward.
"""
from typing import NamedTuple

import torch

from ._ops import ops


class Packed8(NamedTuple):
    """A tensor in 8-bit blocks of 32 values along its last dimension.

    codes : float8_e4m3fn, of the tensor's shape.
    scales : float8_e8m0fnu, [..., ceil(last / 32)], a power of two for each block, 2^-117 to 2^119 (blocks made elsewhere are read
        by the same rule from 2^-117 on; below it small codes are not exact, and the format's NaN scale is not one of them).

    A value is code * scale, within 1/16 of the original's magnitude or 2^-17 of its block's largest,
    whichever is more. It is exact in bfloat16 and float32. NaN and infinities become NaN.
    """
    codes: torch.Tensor
    scales: torch.Tensor


def pack8(x: torch.Tensor) -> Packed8:
    """``x`` (float32, float16 or bfloat16, on a HIP device) in 8-bit blocks. Not differentiable.

    Each block's scale 2^e has the smallest e in [-117, 119] with max |v| <= 448 * 2^e; codes are
    rounded to nearest even.
    """
    return Packed8(*ops.pack8(x))


def unpack8(packed: Packed8, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of ``packed`` (exact in float32 and bfloat16; rounded, and saturated at 65504, in float16)."""
    return ops.unpack8(packed.codes, packed.scales, dtype)


class _Checkpoint8(torch.autograd.Function):
    # Returns the module's output, and x where the module wrote to an x that needs a gradient.
    @staticmethod
    def forward(ctx, module, state, x, *params):
        packed = pack8(x)  # before the module, which may write to x
        version = None if x.is_inference() else x._version
        # Both runs go past autocast's cache of cast weights: it would keep this one's, which carry no gradient, for
        # the rerun and for whoever uses the weights next in the same region.
        ctx.autocast = dict(enabled=torch.is_autocast_enabled("cuda"), dtype=torch.get_autocast_dtype("cuda"), cache_enabled=False)
        with torch.no_grad(), torch.autocast("cuda", **ctx.autocast):
            out = module(x)
        if not isinstance(out, torch.Tensor):
            raise TypeError(f"checkpoint8 takes a module that returns one tensor, not {type(out).__name__}")
        ctx.module, ctx.state, ctx.dtype = module, state, x.dtype
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*packed, *params)
        if not ctx.needs_input_grad[2] or version is None or x._version == version:
            return out
        ctx.mark_dirty(x)
        return x if out is x else (out, x)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, grad_x=None):
        codes, scales, *params = ctx.saved_tensors
        x = unpack8(Packed8(codes, scales), ctx.dtype).requires_grad_(ctx.needs_input_grad[2])
        devices = [x.device] if ctx.state is not None and x.is_cuda else []
        with torch.random.fork_rng(devices, enabled=ctx.state is not None, device_type="cuda"), torch.enable_grad(), \
                torch.autocast("cuda", **ctx.autocast):
            if ctx.state is not None:
                torch.set_rng_state(ctx.state[0])
                for device, state in zip(devices, ctx.state[1:]):
                    torch.cuda.set_rng_state(state, device)
            given = torch.ops.aten._unsafe_view(x, x.shape)  # neither a leaf nor a view to autograd: the module may write to it
            out = ctx.module(given)
        results = [(t, g) for t, g in ((out, grad), (given, grad_x)) if g is not None and t.requires_grad]
        if not results:  # they depend on none of the inputs
            return (None,) * len(ctx.needs_input_grad)
        wanted = [t for t, need in zip([x, *params], ctx.needs_input_grad[2:]) if need]
        grads = iter(torch.autograd.grad([t for t, _ in results], wanted, [g for _, g in results], allow_unused=True))
        return None, None, *(next(grads) if need else None for need in ctx.needs_input_grad[2:])


def checkpoint8(module: torch.nn.Module, x: torch.Tensor, preserve_rng: bool = True) -> torch.Tensor:
    """``module(x)``, keeping only ``x``, in 8 bits, for the backward, which runs the module again on the
    values kept and takes the gradients there.

    The output is the module's own. The gradients are those of the module at the kept values (see
    :class:`Packed8` for how far these are from ``x``). Modules that draw random numbers (dropout, weight noise) draw the
    same ones again, in training or not, from torch's default generators of the CPU and of x's device.
    A module with state that its forward changes (running statistics) changes it twice. A module may write to its
    input in place (torch refuses that for a view that needs a gradient: clone it first); an ``x`` that needs no
    gradient then has the module's values, but no gradient of its parameters through them.

    module : a module of one tensor to one tensor; its parameters' gradients flow as without the checkpoint.
    x : float32, float16 or bfloat16 on a HIP device (any shape the module takes; blocks run along the last dimension).
    preserve_rng : False for a module that draws nothing saves the generators' states. They cannot be read while a
        graph is captured, so a captured step has to pass False.
    """
    params = [p for p in module.parameters() if p.requires_grad]
    if not torch.is_grad_enabled() or not (x.requires_grad or params):
        return module(x)
    state = None
    if preserve_rng:
        if x.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("checkpoint8: the generators' states cannot be read while a graph is captured; pass preserve_rng=False "
                               "for a module that draws no random numbers")
        state = (torch.get_rng_state(), *([torch.cuda.get_rng_state(x.device)] if x.is_cuda else []))
    out = _Checkpoint8.apply(module, state, x, *params)
    return out if isinstance(out, torch.Tensor) else out[0]
