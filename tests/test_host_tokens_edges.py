"""The token-mixing operators without a GPU: layouts and calls that are refused, and the module's arguments."""
import ctypes

import pytest
import torch

import morphocore_amd as mca
from morphocore_amd import _native
from morphocore_amd._native import Heads

F = mca.functional
P = 4096  # a non-null pointer that no refused call follows


def step(state, slots=None):
    batch = 3
    return F.linear_attention_step(torch.zeros(batch, 4, 8), torch.zeros(batch, 2, 8), torch.zeros(batch, 2, 6), torch.zeros(4), state, slots)


# Strides of states [3, 4, 8, 6] (48 values of a head): slots and heads that share memory, and some that don't.
SHARED = [(48, 48), (60, 48), (96, 48), (191, 48), (48, 60), (48, 143), (0, 48), (192, 0), (192, 47), (47, 192)]
APART = [(192, 48), (200, 50), (48, 144), (50, 150), (1000, 48), (384, 96)]


@pytest.mark.parametrize("slot,head", SHARED)
def test_step_refuses_states_that_share_memory(slot, head):
    with pytest.raises(RuntimeError, match="must be dense"):
        step(torch.zeros(8000).as_strided((3, 4, 8, 6), (slot, head, 6, 1)))


@pytest.mark.parametrize("slot,head", APART)
def test_step_takes_states_that_lie_apart(slot, head):
    with pytest.raises(RuntimeError, match="runs on AMD GPUs"):  # what is left to refuse
        step(torch.zeros(8000).as_strided((3, 4, 8, 6), (slot, head, 6, 1)))
    for one in (torch.zeros(1, 4, 8, 6), torch.zeros(8000).as_strided((1, 4, 8, 6), (0, 48, 6, 1))):
        with pytest.raises(RuntimeError, match="runs on AMD GPUs"):
            step(one, torch.zeros(3, dtype=torch.int32))


def test_abi_step_refuses_states_that_share_memory():
    lib = _native.lib()

    def call(slot_stride, head_stride, slots=3, batch=3, heads=4):
        rows = [ctypes.byref(Heads(P, 0, 64, 8, n)) for n in (heads, heads // 2, heads // 2)]
        rc = lib.mca_linear_attention_step(0, *rows, P, P, slot_stride, head_stride, P, 0, slots, P, batch, 8, 6, 1.0, None)
        return rc, lib.mca_last_error().decode()

    for slot, head in SHARED + [(2**40, 2**40), (2**62, 2**62), (2**62, 2**61)]:
        rc, message = call(slot, head)
        assert rc == 1 and ("share memory" in message or "head_stride" in message), (slot, head, message)


def test_step_refuses_an_inference_tensor_outside_of_inference_mode():
    """Before anything is launched: the state would be updated, and the result lost in the error."""
    with torch.inference_mode():
        state = torch.zeros(3, 4, 8, 6)
        with pytest.raises(RuntimeError, match="runs on AMD GPUs"):
            step(state)
    with pytest.raises(RuntimeError, match="inference tensor"):
        step(state)
