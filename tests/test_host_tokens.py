"""The token-mixing operators without a GPU: argument checks of the operators, and the C ABI of
include/morphocore_amd_tokens.h (its symbols, and the refusals that come before any HIP call)."""
import ctypes
import os
import re

import pytest
import torch

import morphocore_amd as mca
from morphocore_amd import _native
from morphocore_amd._native import Heads, Rotation, Sequences

F = mca.functional
HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "morphocore_amd_tokens.h")
P = 4096  # a non-null pointer that no refused call follows


def refused(rc, message):
    assert rc == 1 and message in _native.lib().mca_last_error().decode()


def test_library_exports_every_declared_symbol():
    declared = sorted(set(re.findall(r"\b(mca_\w+)\s*\(", open(HEADER).read())))
    assert sorted(_native.TOKENS_EXPORTS) == declared
    for name in declared:
        assert hasattr(_native.lib(), name), name


def tokens(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def rotary(x=None, positions=None, frequencies=None):
    return F.axial_rotary(tokens(2, 6, 3, 16) if x is None else x, tokens(6, 2, dtype=torch.int32) if positions is None else positions,
                          tokens(2, 8, dtype=torch.float64) if frequencies is None else frequencies)


def normed(q=None, k=None, qw=None, kw=None, eps=1e-6):
    return F.rms_norm_rotary(tokens(6, 3, 16) if q is None else q, tokens(6, 1, 16) if k is None else k, tokens(16) if qw is None else qw,
                             tokens(16) if kw is None else kw, tokens(6, 2, dtype=torch.int32), tokens(2, 8, dtype=torch.float64), eps)


def attention(q=None, k=None, v=None, g=None, state=None, offsets=None):
    return F.linear_attention(tokens(2, 5, 4, 8) if q is None else q, tokens(2, 5, 2, 8) if k is None else k, tokens(2, 5, 2, 6) if v is None else v,
                              tokens(4) if g is None else g, state, offsets)


def step(q=None, k=None, v=None, g=None, state=None, slots=None):
    return F.linear_attention_step(tokens(3, 4, 8) if q is None else q, tokens(3, 2, 8) if k is None else k, tokens(3, 2, 6) if v is None else v,
                                   tokens(4) if g is None else g, tokens(3, 4, 8, 6) if state is None else state, slots)


def test_cpu_tensors_are_refused():
    for call in (rotary, normed, attention, step):
        with pytest.raises(RuntimeError, match="runs on AMD GPUs"):
            call()


@pytest.mark.parametrize("query", [(5, 4, 8), (4, 8), (2, 5, 4, 8, 1)])
def test_attention_ranks(query):
    with pytest.raises(RuntimeError, match=r"query must be \[batch, tokens, heads, values\]"):
        attention(q=tokens(*query))


def test_ranks():
    with pytest.raises(RuntimeError, match=r"with offsets query must be \[tokens, heads, values\]"):
        attention(offsets=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match=r"query must be \[batch, heads, values\]"):
        step(q=tokens(4, 8))
    with pytest.raises(RuntimeError, match=r"must be \[.., heads, values\]"):
        rotary(x=tokens(16))


def test_operator_argument_errors():
    f64, i32 = torch.float64, torch.int32
    leaf = torch.zeros(4, requires_grad=True)
    for call, message in (
            (lambda: rotary(x=tokens(2, 6, 3, 16, dtype=f64)), "not implemented for 'Double'"),
            (lambda: rotary(positions=tokens(6, 2, dtype=f64)), "positions must be int32, int64 or float32"),
            (lambda: rotary(positions=tokens(6, 3, dtype=i32)), "positions must be"),
            (lambda: rotary(positions=tokens(5, 2, dtype=i32)), "positions must be"),
            (lambda: rotary(positions=tokens(1, 6, 2, dtype=i32)), "positions must be"),
            (lambda: rotary(positions=torch.tensor(1, dtype=i32)), "positions must be"),
            (lambda: rotary(frequencies=tokens(2, 8)), "frequencies must be float64"),
            (lambda: rotary(frequencies=tokens(8, dtype=f64)), "frequencies must be float64"),
            (lambda: rotary(frequencies=tokens(2, 9, dtype=f64)), "9 pairs need at least 18 values"),
            (lambda: rotary(frequencies=tokens(2, 8, dtype=f64).requires_grad_()), "have no gradient"),
            (lambda: rotary(positions=tokens(6, 2).requires_grad_()), "have no gradient"),
            (lambda: normed(k=tokens(5, 1, 16)), "key must be"),
            (lambda: normed(k=tokens(6, 1, 15)), "key must be"),
            (lambda: normed(k=tokens(6, 16)), "key must be"),
            (lambda: normed(k=tokens(6, 1, 16, dtype=torch.float16)), "expected scalar type Float"),
            (lambda: normed(qw=tokens(15)), r"weights must be \[16\]"),
            (lambda: normed(kw=tokens(1, 16)), r"weights must be \[16\]"),
            (lambda: normed(kw=tokens(16, dtype=torch.float16)), "expected scalar type Float"),
            (lambda: normed(eps=-1.0), "eps must be non negative"),
            (lambda: normed(eps=float("nan")), "eps must be non negative"),
            (lambda: attention(q=tokens(2, 5, 4, 8, dtype=f64)), "not implemented for 'Double'"),
            (lambda: attention(k=tokens(2, 5, 2, 7)), "key must have"),
            (lambda: attention(k=tokens(2, 4, 2, 8)), "key must have"),
            (lambda: attention(v=tokens(2, 5, 1, 6)), "value must have"),
            (lambda: attention(v=tokens(2, 5, 2, 6, dtype=torch.float16)), "expected scalar type Float"),
            (lambda: attention(k=tokens(2, 5, 3, 8), v=tokens(2, 5, 3, 6)), "must be a multiple"),
            (lambda: attention(k=tokens(2, 5, 0, 8), v=tokens(2, 5, 0, 6)), "must be a multiple"),
            (lambda: attention(g=tokens(2)), r"log_decay must be float32 \[4\]"),
            (lambda: attention(g=tokens(4, dtype=f64)), r"log_decay must be float32 \[4\]"),
            (lambda: attention(g=leaf), "log_decay has no gradient"),
            (lambda: attention(state=tokens(2, 4, 6, 8)), "state must be float32"),
            (lambda: attention(state=tokens(2, 4, 8, 6, dtype=torch.float16)), "state must be float32"),
            (lambda: attention(q=tokens(5, 4, 8), k=tokens(5, 2, 8), v=tokens(5, 2, 6), offsets=torch.zeros(3)), "offsets must be int32 or int64"),
            (lambda: attention(q=tokens(5, 4, 8), k=tokens(5, 2, 8), v=tokens(5, 2, 6), offsets=torch.zeros(1, 3, dtype=i32)), "offsets must be int32 or int64"),
            (lambda: attention(q=tokens(5, 4, 8), k=tokens(5, 2, 8), v=tokens(5, 2, 6), offsets=torch.zeros(0, dtype=i32)), "one entry more"),
            (lambda: step(state=tokens(4, 4, 8, 6)), "without slots state must have 3 entries"),
            (lambda: step(state=tokens(3, 4, 8, 5)), "state must be float32"),
            (lambda: step(state=tokens(3, 4, 8, 6, dtype=torch.bfloat16)), "state must be float32"),
            (lambda: step(state=tokens(3, 4, 6, 8).transpose(2, 3)), "must be dense"),
            (lambda: step(state=tokens(1, 4, 8, 6).expand(3, 4, 8, 6)), "must be dense"),
            (lambda: step(state=tokens(3, 1, 8, 6).expand(3, 4, 8, 6)), "must be dense"),
            (lambda: step(slots=torch.zeros(2, dtype=i32)), r"slots must be \[3\]"),
            (lambda: step(slots=torch.zeros(3)), "slots must be int32 or int64"),
            (lambda: step(q=tokens(3, 4, 8).requires_grad_()), "has no gradient"),
            (lambda: step(state=tokens(3, 4, 8, 6).requires_grad_()), "has no gradient")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: rotary(x=dual(tokens(2, 6, 3, 16))), lambda: normed(qw=dual(tokens(16))), lambda: attention(v=dual(tokens(2, 5, 2, 6))),
                     lambda: attention(state=dual(tokens(2, 4, 8, 6))), lambda: step(k=dual(tokens(3, 2, 8)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_frequencies_and_positions():
    f = F.rotary_frequencies([2, 3], 100.0)
    assert f.dtype == torch.float64 and f.shape == (2, 5)
    want = torch.tensor([[1, 100.0**-0.5, 0, 0, 0], [0, 0, 1, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]], dtype=torch.float64)
    assert torch.allclose(f, want, rtol=1e-15)
    f = F.rotary_frequencies([2, 3], 100.0, shared=True)
    assert torch.allclose(f.sum(0), 100.0 ** (-torch.arange(5, dtype=torch.float64) / 5)) and not f[0, 2:].any() and not f[1, :2].any()
    assert F.rotary_frequencies([0, 1]).shape == (2, 1) and F.rotary_frequencies([0]).shape == (1, 0)
    p = F.grid_positions([2, 3])
    assert p.dtype == torch.int32 and p.tolist() == [[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]
    assert F.grid_positions([4]).tolist() == [[0], [1], [2], [3]] and F.grid_positions([0, 3]).shape == (0, 2)
    for bad in (lambda: F.rotary_frequencies([]), lambda: F.rotary_frequencies([3, -1]), lambda: F.grid_positions([])):
        with pytest.raises(ValueError):
            bad()


def heads(n, data=P, strides=(0, 64, 8)):
    return ctypes.byref(Heads(data, *strides, n))


def rotation(position_type=0, rows=4, axes=2, pairs=4, positions=P, frequencies=P):
    return ctypes.byref(Rotation(positions, position_type, rows, axes, pairs, frequencies, 0))


def test_abi_refuses_rotations():
    lib = _native.lib()

    def call(dtype=0, x=None, out=P, n=4, dim=8, r=None):
        return lib.mca_axial_rotary(dtype, x or heads(2), out, n, dim, r or rotation(), 0, None)

    refused(call(dtype=3), "Unknown dtype")
    refused(call(dim=0), "dim must be")
    refused(call(dim=513), "dim must be")
    refused(call(r=rotation(position_type=3)), "position_type")
    refused(call(r=rotation(axes=0)), "axes must be")
    refused(call(r=rotation(axes=9)), "axes must be")
    refused(call(r=rotation(pairs=5)), "pairs must be")
    refused(call(r=rotation(pairs=-1)), "pairs must be")
    refused(call(r=rotation(rows=0)), "positions must have rows")
    refused(call(r=rotation(positions=None)), "must not be null")
    refused(call(r=rotation(frequencies=None)), "must not be null")
    refused(call(x=heads(-1)), "non negative")
    refused(call(x=heads(2, strides=(0, -1, 8))), "strides must be non negative")
    refused(call(x=heads(2, data=None)), "must not be null")
    refused(call(out=None), "out must not be null")
    refused(call(n=2**60), "too large")
    refused(lib.mca_axial_rotary(0, None, P, 4, 8, rotation(), 0, None), "must not be null")
    refused(lib.mca_axial_rotary(0, heads(2), P, 4, 8, None, 0, None), "must not be null")

    def norm(weight_dtype=0, k=None, qw=P, eps=1e-6, out_k=P):
        return lib.mca_rms_norm_rotary_forward(0, weight_dtype, heads(2), k or heads(1), qw, P, eps, P, out_k, 4, 8, rotation(), None)

    refused(norm(weight_dtype=1), "weight_dtype")
    refused(norm(eps=-1.0), "eps")
    refused(norm(eps=float("nan")), "eps")
    refused(norm(qw=None), "must not be null")
    refused(norm(out_k=None), "must not be null")
    refused(norm(k=heads(65537, strides=(0, 0, 0))), "at most 65536 heads")
    refused(call(x=heads(65537, strides=(0, 0, 0))), "at most 65536 heads")
    need = lib.mca_rms_norm_rotary_backward_workspace_size(4, 3, 8, 4)
    assert need > 0 and lib.mca_rms_norm_rotary_backward_workspace_size(0, 3, 8, 4) == 0
    assert lib.mca_rms_norm_rotary_backward_workspace_size(4, 3, 513, 4) == 0
    assert lib.mca_rms_norm_rotary_backward_workspace_size(10**9, 64, 128, 64) <= 2 * 128 * 4 * 4096

    def back(gk=None, ws=P, size=need, gw=P):
        return lib.mca_rms_norm_rotary_backward(0, 0, heads(2), gk or heads(1), heads(2), heads(1), P, P, 1e-6, P, P, gw, 4, 8, rotation(), ws, size, None)

    refused(back(size=need - 1), "Workspace too small")
    refused(back(ws=None), "Workspace too small")
    refused(back(gk=heads(2)), "must have its tensor's heads")


def sequences(count=2, n=5, offsets=None):
    return ctypes.byref(Sequences(offsets, 0, count, n))


def test_abi_refuses_attention():
    lib = _native.lib()

    def call(dtype=0, s=None, q=None, k=None, v=None, g=P, out=P, dim=8, dv=8, ws=P, size=1 << 40):
        return lib.mca_linear_attention_forward(dtype, s or sequences(), q or heads(4), k or heads(2), v or heads(2), g, None, out, None, dim, dv, 1.0, ws,
                                                size, None)

    refused(call(dtype=-1), "Unknown dtype")
    refused(call(s=sequences(count=-1)), "non negative")
    refused(call(s=sequences(n=-1)), "non negative")
    refused(call(s=sequences(count=2**31)), "Too many sequences")
    refused(call(s=sequences(n=2**62)), "too large")
    refused(call(dim=0), "from 1 to 256")
    refused(call(dim=257), "from 1 to 256")
    refused(call(dv=257), "from 1 to 256")
    refused(call(k=heads(3), v=heads(3)), "multiple")
    refused(call(k=heads(0), v=heads(0)), "multiple")
    refused(call(v=heads(4)), "same heads")
    refused(call(q=heads(4, data=None)), "must not be null")
    refused(call(g=None), "must not be null")
    refused(call(out=None), "must not be null")
    refused(call(q=heads(4, strides=(0, 8, -8))), "strides")
    refused(lib.mca_linear_attention_forward(0, None, heads(4), heads(2), heads(2), P, None, P, None, 8, 8, 1.0, P, 1 << 40, None), "must not be null")
    long = sequences(1, 10**6)
    need = lib.mca_linear_attention_forward_workspace_size(2, long, 4, 128, 128)
    if need:
        refused(call(dtype=2, s=long, dim=128, dv=128, size=need - 1), "Workspace too small")
    assert lib.mca_linear_attention_forward_workspace_size(2, long, 4, 128, 257) == 0

    def back(go=None, g=P, size=1 << 40, ws=P, k=None):
        return lib.mca_linear_attention_backward(0, sequences(), go or heads(4), None, heads(4), k or heads(2), heads(2), g, None, P, P, P, P, 8, 8, 1.0, ws,
                                                 size, None)

    refused(back(go=heads(2)), "same heads")
    refused(back(g=None), "log_decay")
    need = lib.mca_linear_attention_backward_workspace_size(0, sequences(), 4, 2, 8, 8)
    assert need > 0  # the float32 gradients of the shared heads
    refused(back(size=need - 1), "Workspace too small")
    refused(back(ws=None), "Workspace too small")

    def step(slots=3, batch=3, slot_of=None, slot_stride=4 * 64, head_stride=64, states=P, k=None):
        return lib.mca_linear_attention_step(0, heads(4), k or heads(2), heads(2), P, states, slot_stride, head_stride, slot_of, 0, slots, P, batch, 8, 8,
                                             1.0, None)

    refused(step(slots=2), "a slot for every sequence")
    refused(step(head_stride=63), "head_stride")
    refused(step(slot_stride=-1), "slot_stride")
    refused(step(states=None), "must not be null")
    refused(step(k=heads(3)), "multiple")


def test_attention_workspace_does_not_grow_with_short_sequences():
    lib = _native.lib()
    for dtype in range(3):
        for count, n in [(41, 12001), (10**4, 10**5), (10**6, 10**6), (64, 32768), (3, 10**7)]:
            size = lib.mca_linear_attention_forward_workspace_size(dtype, sequences(count, n, P), 16, 128, 128)
            # At most the state of every 64 tokens.
            assert size <= 16 * 128 * 128 * 4 * (n // 64) + 256, (dtype, count, n)
            if n <= 100 * count:
                assert size == 0, (dtype, count, n)


# ------------------------------------------------------------------------------------------------
# The module
# ------------------------------------------------------------------------------------------------

def test_token_mixer():
    m = mca.nn.TokenMixer(48, 4, axes=3, kv_heads=2, eps=1e-5)
    shapes = {k: tuple(v.shape) for k, v in m.state_dict().items()}
    assert shapes == {"norm.weight": (48,), "query_weight": (12,), "key_weight": (12,), "project": (96, 48), "contract": (48, 48), "log_decay": (4,)}
    assert m.norm.eps == 1e-5 and m.frequencies.shape == (3, 6) and bool((m.frequencies.ne(0).sum(1) == 2).all())
    # Decays and frequencies are as they were whatever the module's type becomes.
    decay, frequencies = m.log_decay.clone(), m.frequencies.clone()
    for t in (torch.bfloat16, torch.float64, torch.float32):
        m = m.to(t)
        assert m.project.dtype == t and torch.equal(m.log_decay, decay) and m.log_decay.dtype == torch.float32
        assert torch.equal(m.frequencies, frequencies) and m.frequencies.dtype == torch.float64
    assert torch.allclose(-1 / decay, torch.tensor([16.0, 16.0 * 2**(8 / 3), 16.0 * 2**(16 / 3), 4096.0]))
    assert mca.nn.TokenMixer(8, 1).log_decay.tolist() == [-1 / 16] and mca.nn.TokenMixer(8, 2, dim=7).frequencies.shape == (1, 3)
    for bad in (lambda: mca.nn.TokenMixer(0, 1), lambda: mca.nn.TokenMixer(8, 0), lambda: mca.nn.TokenMixer(8, 4, kv_heads=3),
                lambda: mca.nn.TokenMixer(8, 4, axes=2), lambda: mca.nn.TokenMixer(8, 1, axes=0), lambda: mca.nn.TokenMixer(8, 2, kv_heads=0),
                lambda: mca.nn.TokenMixer(257, 1), lambda: mca.nn.TokenMixer(64, 1, axes=9)):
        with pytest.raises(ValueError):
            bad()
