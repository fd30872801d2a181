"""The channel-mixing operators without a GPU: argument checks of the operators, and the C ABI of
include/morphocore_amd_mixer.h (its symbols, and the refusals that come before any HIP call)."""
import os
import re

import pytest
import torch

import morphocore_amd as mca
from morphocore_amd import _native

F = mca.functional
HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "morphocore_amd_mixer.h")
P = 4096  # a non-null pointer that no refused call follows


def refused(rc, message):
    assert rc == 1 and message in _native.lib().mca_last_error().decode()


def test_library_exports_every_declared_symbol():
    declared = sorted(set(re.findall(r"\b(mca_\w+)\s*\(", open(HEADER).read())))
    assert sorted(_native.MIXER_EXPORTS) == declared
    for name in declared:
        assert hasattr(_native.lib(), name), name


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(3, 64), torch.ones(64)
    p = F.Packed8(torch.zeros(3, 64).to(torch.float8_e4m3fn), torch.ones(3, 2).to(torch.float8_e8m0fnu))
    for call in (lambda: F.pack8(x), lambda: F.unpack8(p), lambda: F.rms_norm(x, w), lambda: F.rms_norm8(x, w), lambda: F.gated_silu(x),
                 lambda: F.gated_silu8(x, x), lambda: F.linear8(x, torch.zeros(5, 64)), lambda: F.grad_weight8(torch.zeros(3, 5), p)):
        with pytest.raises(RuntimeError, match="runs on AMD GPUs"):
            call()


def test_operator_argument_errors():
    x, w = torch.zeros(3, 64), torch.ones(64)
    for call, message in (
            (lambda: F.pack8(torch.tensor(1.0)), "at least one dimension"),
            (lambda: F.rms_norm(x, torch.ones(63)), r"weight must be \[64\]"),
            (lambda: F.rms_norm(x, torch.ones(1, 64)), r"weight must be \[64\]"),
            (lambda: F.rms_norm(x, w, eps=-1.0), "eps must be non negative"),
            (lambda: F.rms_norm(x, w, eps=float("nan")), "eps must be non negative"),
            (lambda: F.linear8(x, torch.ones(5, 63)), r"weight must be \[out, 64\]"),
            (lambda: F.linear8(x, torch.ones(64)), r"weight must be \[out, 64\]"),
            (lambda: F.unpack8(F.Packed8(x, x)), "codes must be float8_e4m3fn"),
            (lambda: F.unpack8(F.Packed8(x.to(torch.float8_e4m3fn), x)), "scales must be float8_e8m0fnu"),
            (lambda: F.unpack8(F.Packed8(x.to(torch.float8_e4m3fn), torch.ones(3, 1).to(torch.float8_e8m0fnu))), "need scales of shape"),
            (lambda: torch.ops.morphocore.linear8(x, torch.ones(5, 64), x), "codes and scales go together")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_abi_refuses_types_sizes_and_strides():
    lib = _native.lib()
    refused(lib.mca_pack8(3, P, 8, P, P, 4, 8, None), "Unknown dtype")
    refused(lib.mca_pack8(-1, P, 8, P, P, 4, 8, None), "Unknown dtype")
    refused(lib.mca_pack8(0, P, 8, P, P, -4, 8, None), "non negative")
    refused(lib.mca_pack8(0, P, 8, P, P, 4, 2**31, None), "below 2^31")
    refused(lib.mca_pack8(0, P, 8, P, P, 2**62, 2**20, None), "too large")
    refused(lib.mca_pack8(0, P, -8, P, P, 4, 8, None), "strides must be non negative")
    refused(lib.mca_pack8(0, None, 8, P, P, 4, 8, None), "must not be null")
    refused(lib.mca_unpack8(0, P, None, P, 4, 8, None), "must not be null")
    refused(lib.mca_rms_norm_forward(1, 2, P, 8, None, 0, P, 1e-6, P, None, None, None, None, 4, 8, None), "weight_dtype")
    refused(lib.mca_rms_norm_forward(0, 0, P, 8, None, 0, P, -1.0, P, None, None, None, None, 4, 8, None), "eps")
    refused(lib.mca_rms_norm_forward(0, 0, P, 8, None, 0, P, 0.0, P, None, P, None, None, 4, 8, None), "go together")
    refused(lib.mca_rms_norm_forward(0, 0, P, 8, None, 0, None, 0.0, P, None, None, None, None, 4, 8, None), "must not be null")
    refused(lib.mca_rms_norm_backward(0, 0, P, 8, None, 0, P, 8, P, P, P, P, 4, 8, None, 0, None), "Workspace too small")
    refused(lib.mca_rms_norm_backward(0, 0, P, 8, None, 0, P, 8, P, None, P, None, 4, 8, None, 0, None), "must not be null")
    refused(lib.mca_gated_silu_forward(0, P, 8, None, 8, P, None, None, None, None, None, None, 4, 8, None), "must not be null")
    refused(lib.mca_gated_silu_forward(0, P, 8, P, 8, P, P, None, None, None, None, None, 4, 8, None), "go together")
    refused(lib.mca_gated_silu_backward(0, P, 8, P, 8, None, 8, None, None, None, None, P, P, 8, 4, 8, None), "go together")
    refused(lib.mca_gated_silu_backward(0, P, 8, None, 8, None, 8, P, P, P, None, P, P, 8, 4, 8, None), "packed form")
    refused(lib.mca_gated_silu_backward(0, P, 8, P, 8, P, 8, None, None, None, None, P, P, 7, 4, 8, None), "grad_stride")
    refused(lib.mca_grad_weight8(0, 1, P, 8, P, P, P, 4, 8, 8, P, 1 << 20, None), "weight_dtype")
    need = lib.mca_grad_weight8_workspace_size(0, 100000, 64, 64)  # rows in splits
    assert need > 0
    refused(lib.mca_grad_weight8(0, 0, P, 64, P, P, P, 100000, 64, 64, P, need - 1, None), "Workspace too small")
    refused(lib.mca_grad_weight8(0, 0, P, 64, P, P, P, 100000, 64, 64, None, need, None), "Workspace too small")
    refused(lib.mca_grad_weight8(0, 0, P, 8, P, P, None, 4, 8, 8, P, 1 << 20, None), "must not be null")


def test_abi_workspace_sizes():
    lib = _native.lib()
    assert lib.mca_rms_norm_backward_workspace_size(0, 64) == 0 and lib.mca_rms_norm_backward_workspace_size(1, 64) >= 256
    assert lib.mca_grad_weight8_workspace_size(0, 0, 64, 64) == 0 and lib.mca_grad_weight8_workspace_size(9, 8, 64, 64) == 0
    # A few times the sums' own size however many rows are summed.
    for rows in (1, 1000, 10**6, 10**9):
        assert lib.mca_rms_norm_backward_workspace_size(rows, 4096) <= 4096 * 4 * 1024
        assert lib.mca_grad_weight8_workspace_size(2, rows, 64, 64) <= 64 * 64 * 4 * 1024


def test_modules():
    m = mca.nn.ChannelMixer(48, 80, eps=1e-5)
    shapes = {k: tuple(v.shape) for k, v in m.state_dict().items()}
    assert shapes == {"norm.weight": (48,), "expand": (160, 48), "contract": (48, 80)}
    assert torch.equal(m.norm.weight, torch.ones(48)) and m.norm.eps == 1e-5
    assert mca.nn.Checkpoint8(torch.nn.Linear(3, 4)).module.weight.shape == (4, 3)
    for bad in (lambda: mca.nn.ChannelMixer(0, 8), lambda: mca.nn.ChannelMixer(8, 0), lambda: mca.nn.RMSNorm(0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        mca.nn.Checkpoint8(torch.tanh)
