"""The C ABI and the operators of channel mixing without a GPU: calls that launch nothing."""
from morphocore_amd import _native

P = 4096  # a non-null pointer that no call follows


def test_backward_of_a_gated_activation_without_rows():
    """gate is an empty array's null pointer, up the address of its second half: nothing is read of either."""
    lib = _native.lib()
    for gate, up in ((None, P), (P, None), (None, None), (P, P)):
        assert lib.mca_gated_silu_backward(0, P, 8, gate, 16, up, 16, None, None, None, None, P, P, 16, 0, 8, None) == 0
