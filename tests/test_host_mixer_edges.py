"""The C ABI and the operators of channel mixing without a GPU: calls that launch nothing."""
import pytest
import torch
import torch.autograd.forward_ad as forward

import morphocore_amd.functional as F
from morphocore_amd import _native

P = 4096  # a non-null pointer that no call follows


def test_backward_of_a_gated_activation_without_rows():
    """gate is an empty array's null pointer, up the address of its second half: nothing is read of either."""
    lib = _native.lib()
    for gate, up in ((None, P), (P, None), (None, None), (P, P)):
        assert lib.mca_gated_silu_backward(0, P, 8, gate, 16, up, 16, None, None, None, None, P, P, 16, 0, 8, None) == 0


@pytest.mark.parametrize("call,operands", [(lambda x, w, u: F.rms_norm(x, w), 2), (lambda x, w, u: F.rms_norm(x, w, u), 3),
                                           (lambda x, w, u: F.rms_norm8(x, w, u), 3), (lambda g, u, _: F.gated_silu(g), 1),
                                           (lambda g, u, _: F.gated_silu(g, u), 2), (lambda g, u, _: F.gated_silu8(g), 1),
                                           (lambda g, u, _: F.gated_silu8(g, u), 2)])
def test_forward_mode_derivatives_are_refused(call, operands):
    """Not lost: without a gradient to record the operators write into new tensors, which have no tangent."""
    tensors = [torch.randn(64) for _ in range(3)]
    for at in range(operands):
        with forward.dual_level():
            args = list(tensors)
            args[at] = forward.make_dual(args[at], torch.ones(64))
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call(*args)
            with forward._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="runs on AMD GPUs"):
                call(*args)
    with pytest.raises(RuntimeError, match="runs on AMD GPUs"):
        call(*tensors)
