"""The token-mixing operators on the GPU against the float64 oracle (tests/tokens_oracle.py).

Tolerances, with u the unit roundoff of the output's type (2^-24, 2^-11, 2^-8) and f = 2^-24:
Rotation: the fraction of a turn is rounded to float32 (an angle's error of pi 2^-25 < 2 f), sine and cosine to 2 units, a
product and an addition each: 8 f (|a| + |b|). The norm before it adds half of a sum's error (16 terms a lane and 6 levels),
a root, a division and two products, below 24 f of the same; its gradients two such sums and six operations more, 64 f of the terms'
magnitudes; sums over n rows 2 sqrt(n) + 64 units f (the usual growth of a sum's rounding errors).
Attention, of the sum M of the terms' magnitudes (each decay's reach counted into it): products of dim terms and sums over the
tokens, 2 sqrt(dim) + 2 sqrt(tokens) + 64 units f. Outputs of 16 bits may hold scores and states in two terms of 8 bits, to
2^-16 each, and leave out the product of two second terms, 2^-16: 2^-14 M.
Subnormal outputs add half their spacing.
"""
import math

import numpy as np
import pytest
import torch

import morphocore_amd.functional as F
from tests import tokens_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
f32 = 2.0**-24


def np64(t):
    return t.detach().double().cpu().numpy()


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def near(got, want, size, what=""):
    """|got - want| <= size + u |want| + the subnormals' half spacing, elementwise."""
    dtype = got.dtype
    got = np64(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    far = np.abs(got - want)
    bad = ~(far <= size + U[dtype] * np.abs(want) + TINY[dtype])
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values, first {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"


# ------------------------------------------------------------------------------------------------
# Rotations
# ------------------------------------------------------------------------------------------------

# dim, pairs
ROWS = [(1, 0), (2, 1), (5, 2), (8, 3), (16, 8), (24, 7), (33, 16), (40, 3), (64, 32), (72, 33), (80, 40), (100, 9), (128, 64), (200, 90), (256, 128), (257, 13),
        (300, 150), (512, 256), (512, 0)]


def table(axes, pairs, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(axes, pairs, generator=g, dtype=torch.float64) * 2 - 0.3).to(DEV)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", ROWS)
@pytest.mark.parametrize("dtype", TYPES)
def test_rotary(dtype, dim, pairs, interleaved):
    x = randn(dim, 2, 7, 3, dim, dtype=dtype).requires_grad_()
    p, f = torch.randint(-9, 40, (7, 2), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV), table(2, pairs)
    y = F.axial_rotary(x, p, f, interleaved)
    angle = O.angles(p.cpu().numpy(), f.cpu().numpy())
    assert y.dtype == dtype
    near(y, O.rotate(np64(x), angle, interleaved), 8 * f32 * O.pair_size(np64(x), pairs, interleaved), "y")
    assert torch.equal(y[..., 2 * pairs:], x[..., 2 * pairs:])
    gy = randn(dim + 1, *x.shape, dtype=dtype)
    (gx,) = torch.autograd.grad(y, x, gy)
    near(gx, O.rotate(np64(gy), -angle, interleaved), 8 * f32 * O.pair_size(np64(gy), pairs, interleaved), "gx")
    with torch.no_grad():
        assert torch.equal(F.axial_rotary(x, p, f, interleaved), y)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("axes", [1, 3, 8])
def test_rotary_positions(kind, axes):
    """Far positions of every type, for every token or shared by the batch."""
    x = randn(3, 4, 5, 2, 64)
    p = (torch.rand(4, 5, axes, generator=torch.Generator().manual_seed(2), dtype=torch.float64) * 2e6 - 1e6).to(kind)
    f = table(axes, 32, 3)
    for at in (p, p[1]):
        y = F.axial_rotary(x, at.to(DEV), f)
        angle = O.angles(at.double().numpy(), f.cpu().numpy())
        # Beside the float32 errors those of float64 angles up to 8 * 1.7e6.
        near(y, O.rotate(np64(x), angle, False), (8 * f32 + 2.0**-48 * 1e8) * O.pair_size(np64(x), 32, False))
    if kind == torch.int64:
        y = F.axial_rotary(x, torch.full((5, axes), 2**40, device=DEV), torch.full((axes, 32), math.pi, dtype=torch.float64, device=DEV))
        assert torch.isfinite(y).all()


def test_rotary_reads_strided_and_permuted_heads():
    wide, f = randn(4, 3, 6, 5, 200, dtype=torch.bfloat16), table(1, 20)
    p = torch.arange(6, device=DEV, dtype=torch.int32)[:, None]
    for x in (wide[..., 40:90], wide[:, :, 1:4, 3:52], wide[..., ::3], wide[:1].expand(4, 6, 5, 200), wide.transpose(0, 2)[:, :, :, :50], wide[:, :, ::2],
              wide[0], wide[..., :50].transpose(2, 1)[:, :5].transpose(1, 2)):
        assert torch.equal(F.axial_rotary(x, p, f), F.axial_rotary(x.contiguous(), p, f))
    one = wide[0, 0]  # a single token's heads
    assert torch.equal(F.axial_rotary(one, p[3], f), F.axial_rotary(one[None], p[3:4], f)[0])


def test_rotary_many_tokens():
    """More tokens than a launch has groups of lanes, and a batch that shares positions."""
    x, f = randn(5, 9, 30011, 1, 16, dtype=torch.float16), table(2, 8)
    p = F.grid_positions([30011, 1], device=DEV)
    y = F.axial_rotary(x, p, f, True)
    want = O.rotate(np64(x), O.angles(p.cpu().numpy(), f.cpu().numpy()), True)
    near(y, want, (8 * f32 + 2.0**-48 * 1e5) * O.pair_size(np64(x), 8, True))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", ROWS)
@pytest.mark.parametrize("dtype,wtype", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_norm_rotary(dtype, wtype, dim, pairs, interleaved):
    heads, kvh, n = 5, 2, 11
    joint = randn(dim, n, (heads + 2 * kvh) * dim, dtype=dtype, scale=2.0)
    q = joint[:, :heads * dim].unflatten(-1, (heads, dim)).detach().requires_grad_()
    k = joint[:, heads * dim:(heads + kvh) * dim].unflatten(-1, (kvh, dim)).detach().requires_grad_()
    qw, kw = ((1 + randn(s, dim, scale=0.3)).to(wtype).requires_grad_() for s in (7, 8))
    p, f, eps = torch.arange(n, device=DEV)[:, None] * 17 - 40, table(1, pairs, 2), 1e-3
    outs = F.rms_norm_rotary(q, k, qw, kw, p, f, eps, interleaved)
    angle = O.angles(p.cpu().numpy(), f.cpu().numpy())
    gys = [randn(dim + 3, *o.shape, dtype=dtype) for o in outs]
    grads = torch.autograd.grad(outs, [q, k, qw, kw], gys)
    for x, w, y, gy, gx, gw in zip((q, k), (qw, kw), outs, gys, grads[:2], grads[2:]):
        X, W, G = np64(x), np64(w), np64(gy)
        n64 = O.norm(X, W, eps)
        near(y, O.rotate(n64, angle, interleaved), 32 * f32 * O.pair_size(n64, pairs, interleaved), "y")
        wx, ww = O.norm_grads(X, W, eps, O.rotate(G, -angle, interleaved))
        sx, sw = O.norm_sizes(X, W, eps, O.pair_size(G, pairs, interleaved))
        near(gx, wx, 64 * f32 * sx, "gx")
        near(gw, ww, (2 * math.sqrt(X.shape[0] * X.shape[1]) + 64) * f32 * sw, "gw")
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs, F.rms_norm_rotary(q, k, qw, kw, p, f, eps, interleaved)))


@pytest.mark.parametrize("n,heads,kvh", [(1, 40, 8), (70000, 2, 1), (5000, 13, 3), (3, 0, 4), (3, 4, 0), (0, 4, 2), (2500, 64, 16)])
def test_norm_rotary_launches(n, heads, kvh):
    """Few tokens with many heads, many with few, none."""
    q, k, w = randn(1, n, heads, 48, dtype=torch.bfloat16).requires_grad_(), randn(2, n, kvh, 48, dtype=torch.bfloat16).requires_grad_(), randn(3, 48).requires_grad_()
    w2 = randn(4, 48).requires_grad_()
    p, f = torch.arange(n, device=DEV, dtype=torch.int32)[:, None], table(1, 20)
    outs = F.rms_norm_rotary(q, k, w, w2, p, f)
    angle = O.angles(p.cpu().numpy(), f.cpu().numpy())
    gys = [randn(5, *o.shape, dtype=torch.bfloat16) for o in outs]
    grads = torch.autograd.grad(outs, [q, k, w, w2], gys)
    for x, ww, y, gy, gx, gw in zip((q, k), (w, w2), outs, gys, grads[:2], grads[2:]):
        X, W, G = np64(x), np64(ww), np64(gy)
        n64 = O.norm(X, W, 1e-6) if X.size else X
        near(y, O.rotate(n64, angle, False), (32 * f32 + 2.0**-48 * 1e5) * O.pair_size(n64, 20, False), "y")
        if not X.size:
            assert not gw.any()
            continue
        wx, wg = O.norm_grads(X, W, 1e-6, O.rotate(G, -angle, False))
        sx, sw = O.norm_sizes(X, W, 1e-6, O.pair_size(G, 20, False))
        near(gx, wx, (64 * f32 + 2.0**-48 * 1e5) * sx, "gx")
        near(gw, wg, ((2 * math.sqrt(n * X.shape[1]) + 64) * f32 + 2.0**-48 * 1e5) * sw, "gw")


def test_norm_rotary_keeps_rows_apart():
    """Zeros, infinities and NaN in a head's row reach that row alone; rows of zeros give zeros."""
    q, k, w = randn(1, 9, 4, 64), randn(2, 9, 2, 64), torch.ones(64, device=DEV)
    p, f = torch.arange(9, device=DEV)[:, None], table(1, 32)
    clean = F.rms_norm_rotary(q, k, w, w, p, f)
    bad = q.clone()
    bad[2, 1], bad[3, 0, 5], bad[4, 3, 60] = 0.0, float("inf"), float("nan")
    outs = F.rms_norm_rotary(bad, k, w, w, p, f)
    assert not outs[0][2, 1].any() and not torch.isfinite(outs[0][3, 0]).all() and torch.isnan(outs[0][4, 3]).all()
    same = torch.ones(9, 4, dtype=torch.bool)
    same[2, 1] = same[3, 0] = same[4, 3] = False
    assert torch.equal(outs[0][same], clean[0][same]) and torch.equal(outs[1], clean[1])


def test_norm_rotary_missing_gradients():
    q, k, w = randn(1, 9, 4, 32).requires_grad_(), randn(2, 9, 2, 32).requires_grad_(), torch.ones(32, device=DEV, requires_grad=True)
    p, f = torch.arange(9, device=DEV)[:, None], table(1, 10)
    gy = randn(3, 9, 4, 32)
    oq, _ = F.rms_norm_rotary(q, k, w, w.detach(), p, f)
    gq, gk, gw = torch.autograd.grad(oq, [q, k, w], gy)
    both = torch.autograd.grad(F.rms_norm_rotary(q, k, w, w.detach(), p, f), [q, k, w], [gy, torch.zeros_like(k)])
    assert all(torch.equal(a, b) for a, b in zip((gq, gk, gw), both)) and not gk.any()
    (only,) = torch.autograd.grad(F.rms_norm_rotary(q, k.detach(), w.detach(), w.detach(), p, f)[0], [q], gy)
    assert torch.equal(only, gq)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(F.axial_rotary(q, p, f).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(F.rms_norm_rotary(q, k, w, w, p, f)[0].sum(), q, create_graph=True)


# ------------------------------------------------------------------------------------------------
# Linear attention
# ------------------------------------------------------------------------------------------------


def decays(heads):
    """From two tokens' reach to none lost at all, and no memory."""
    g = torch.log1p(-torch.exp2(-torch.linspace(1, 11, heads, dtype=torch.float64))).float()
    if heads > 2:
        g[1] = 0.0
    if heads > 3:
        g[2] = -float("inf")
    return g.to(DEV)


def inputs(seed, rows, heads, kvh, dim, dv, dtype, states=0):
    q, k, v = randn(seed, *rows, heads, dim, dtype=dtype), randn(seed + 1, *rows, kvh, dim, dtype=dtype), randn(seed + 2, *rows, 2 * kvh * dv, dtype=dtype)
    v = v[..., kvh * dv:].unflatten(-1, (kvh, dv))
    go, first, last = randn(seed + 3, *rows, heads, dv, dtype=dtype), randn(seed + 4, states, heads, dim, dv), randn(seed + 5, states, heads, dim, dv)
    return [t.detach().requires_grad_() for t in (q, k, v, first)] + [go, last]


def sizes(dtype, dim, n):
    """Allowed error of outputs of the inputs' type and of states, in units of M."""
    f = (2 * math.sqrt(dim) + 2 * math.sqrt(n) + 64) * f32
    return f if dtype == torch.float32 else f + 2.0**-14, f


def check_sequence(results, q, k, v, g, scale, first, go, last, what):
    """results: name -> tensor of one sequence."""
    n = q.shape[0]
    want = O.attention(np64(q), np64(k), np64(v), np64(g), scale, None if first is None else np64(first), None if go is None else np64(go),
                       None if last is None else np64(last))
    for name, got in results.items():
        if got is None:
            continue
        value, size = want[name]
        out, state = sizes(q.dtype, max(q.shape[-1], v.shape[-1]) * (q.shape[1] // k.shape[1]), n)
        near(got, value, (state if name in ("state", "gs") else out) * size, f"{what} {name}")


LENGTHS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 128, 129, 257]
DIMS = [(1, 1), (3, 7), (16, 16), (32, 32), (33, 20), (64, 64), (40, 100), (128, 128), (96, 77), (65, 129), (128, 256), (256, 64), (256, 256)]


def attend(q, k, v, first, go, last, g, scale, offsets=None):
    out, state = F.linear_attention(q, k, v, g, first, offsets, scale, True)
    assert out.dtype == q.dtype and state.dtype == torch.float32
    grads = torch.autograd.grad([out, state], [q, k, v, first], [go, last])
    return [out, state, *grads]


@pytest.mark.parametrize("dim,dv", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_dims(dtype, dim, dv):
    q, k, v, first, go, last = inputs(dim + dv, (2, 150), 4, 2, dim, dv, dtype, 2)
    g, scale = decays(4), dim**-0.5
    out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, scale)
    for b in range(2):
        check_sequence(dict(out=out[b], state=state[b], gq=gq[b], gk=gk[b], gv=gv[b], gs=gs[b]), q[b], k[b], v[b], g, scale, first[b], go[b], last[b], f"{b}")


@pytest.mark.parametrize("n", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_lengths(dtype, n):
    q, k, v, first, go, last = inputs(n, (3, n), 5, 5, 48, 64, dtype, 3)
    g, scale = decays(5), 0.3
    out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, scale)
    for b in range(3):
        check_sequence(dict(out=out[b], state=state[b], gq=gq[b], gk=gk[b], gv=gv[b], gs=gs[b]), q[b], k[b], v[b], g, scale, first[b], go[b], last[b], f"{b}")
    with torch.no_grad():
        again, end = F.linear_attention(q, k, v, g, first, scale=scale, final_state=True)
        assert torch.equal(again, out) and torch.equal(end, state) and torch.equal(F.linear_attention(q, k, v, g, first, scale=scale), out)
        out = F.linear_attention(q, k, v, g)  # no state, the scale by default
    for b in range(3):
        check_sequence(dict(out=out[b]), q[b], k[b], v[b], g, 48**-0.5, None, None, None, f"{b}")


@pytest.mark.parametrize("heads,kvh", [(1, 1), (4, 1), (6, 3), (8, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_long(dtype, heads, kvh):
    """Sequences long enough to be split over workgroups."""
    n = 2111
    q, k, v, first, go, last = inputs(heads, (1, n), heads, kvh, 64, 64, dtype, 1)
    g, scale = decays(heads), 0.125
    out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, scale)
    check_sequence(dict(out=out[0], state=state[0], gq=gq[0], gk=gk[0], gv=gv[0], gs=gs[0]), q[0], k[0], v[0], g, scale, first[0], go[0], last[0], "")


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_packed(dtype, wide):
    """Packed sequences of none, one and many rows; rows of no sequence, before and behind, hold NaN and get zeros."""
    lengths = [0, 1, 70, 0, 64, 129, 1, 400, 0]
    before, behind = 3, 90
    offsets = torch.tensor([before] + [before + sum(lengths[:i + 1]) for i in range(len(lengths))], dtype=torch.int64 if wide else torch.int32)
    n = int(offsets[-1]) + behind
    q, k, v, first, go, last = inputs(9, (n,), 4, 2, 64, 80, dtype, len(lengths))
    with torch.no_grad():
        for t in (q, k, v, go):
            t[:before], t[int(offsets[-1]):] = float("nan"), float("nan")
    g, scale = decays(4), 0.2
    out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, scale, offsets.to(DEV))
    for t in (out, gq, gk, gv):
        assert not t[:before].any() and not t[int(offsets[-1]):].any()
    for i in range(len(lengths)):
        r = slice(int(offsets[i]), int(offsets[i + 1]))
        check_sequence(dict(out=out[r], state=state[i], gq=gq[r], gk=gk[r], gv=gv[r], gs=gs[i]), q[r], k[r], v[r], g, scale, first[i], go[r], last[i], f"{i}")


def test_attention_offsets_out_of_range():
    """Offsets beyond the rows are taken as the nearest row: nothing outside is touched."""
    q, k, v, first, go, last = inputs(1, (50,), 2, 2, 16, 16, torch.float32, 2)
    wild, tame = torch.tensor([-5, 20, 10**6], device=DEV), torch.tensor([0, 20, 50], device=DEV)
    g = decays(2)
    for a, b in zip(attend(q, k, v, first, go, last, g, 1.0, wild), attend(q, k, v, first, go, last, g, 1.0, tame)):
        assert torch.equal(a, b)


def test_attention_empty():
    g = decays(4)
    for rows, offsets, states in (((0, 5), None, 0), ((2, 0), None, 2), ((0,), torch.tensor([0, 0, 0], device=DEV), 2), ((7,), torch.tensor([7], device=DEV), 0)):
        q, k, v, first, go, last = inputs(1, rows, 4, 2, 16, 8, torch.float32, states)
        out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, 1.0, offsets)
        assert not out.any() and torch.equal(state, first) and torch.equal(gs, last) and not any(t.any() for t in (gq, gk, gv))
        assert out.shape == (*rows, 4, 8) and gk.shape == k.shape
    q, k, v, first, go, last = inputs(1, (2, 5), 0, 0, 16, 8, torch.float32, 2)
    assert F.linear_attention(q, k, v, decays(0)).shape == (2, 5, 0, 8)


def test_attention_many_sequences():
    """More sequences than a grid's second dimension, most of one row."""
    n = 70000
    q, k, v, first, go, last = inputs(2, (n,), 2, 1, 8, 8, torch.bfloat16, n)
    g = decays(2)
    offsets = torch.arange(n + 1, device=DEV, dtype=torch.int32)
    out, state, gq, gk, gv, gs = attend(q, k, v, first, go, last, g, 0.5, offsets)
    d = torch.exp(g.double())[:, None, None]
    s = d * first.double() + k.double().unsqueeze(-1) * v.double().unsqueeze(-2)
    want = 0.5 * (q.double().unsqueeze(-2) @ s).squeeze(-2)
    assert (state - s).abs().max() < 1e-5 and ((out - want).abs() <= 2.0**-8 * want.abs() + 1e-3).all()
    assert (gs - d * (last.double() + 0.5 * q.double().unsqueeze(-1) * go.double().unsqueeze(-2))).abs().max() < 1e-5


def test_attention_more_sequences_than_workgroups():
    """Sequences of one token, which a workgroup takes one after another, a value that is not finite among them."""
    n = 600000
    q, k, v, *_ = inputs(4, (n,), 2, 1, 3, 2, torch.float32, 0)
    q, k, v = q.detach(), k.detach(), v.detach().clone()
    v[123456, 0, 1] = float("inf")
    out = F.linear_attention(q, k, v, decays(2), offsets=torch.arange(n + 1, device=DEV), scale=0.5)
    want = 0.5 * (q.double() * k.double()).sum(-1, keepdim=True) * v.double()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[123456, :, 1] = True
    assert torch.equal(out.isnan(), bad) and ((out - want)[~bad].abs() <= 2.0**-18 * (q.abs() * k.abs()).sum(-1, keepdim=True).mul(v.abs())[~bad]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_packed_segments(dtype):
    """Sequences about a segment's length and several long, which are split and begin where others' segments end."""
    lengths = [130, 1, 127, 128, 129, 700, 0, 63, 257, 256, 255, 3, 900, 64, 385]
    heads, kvh, dim, dv = 2, 1, 32, 16
    q, k, v, first, go, last = inputs(6, (sum(lengths),), heads, kvh, dim, dv, dtype, len(lengths))
    g = decays(heads)
    offsets = torch.tensor([0, *np.cumsum(lengths)], device=DEV)
    names = ["out", "state", "gq", "gk", "gv", "gs"]
    got = dict(zip(names, attend(q, k, v, first, go, last, g, 0.3, offsets)))
    for i, n in enumerate(lengths):
        rows = slice(int(offsets[i]), int(offsets[i + 1]))
        if n:
            check_sequence({x: got[x][i] if x in ("state", "gs") else got[x][rows] for x in names}, q[rows], k[rows], v[rows], g, 0.3, first[i], go[rows],
                           last[i], f"sequence {i}")
        else:
            assert torch.equal(got["state"][i], first[i]) and torch.equal(got["gs"][i], last[i])


def test_attention_strides():
    """Operands in any order of their dimensions, expanded, and behind 32-bit offsets."""
    q, k, v, first, go, last = inputs(3, (2, 70), 4, 4, 32, 32, torch.bfloat16, 2)
    g = decays(4)
    want = attend(q, k, v, first, go, last, g, 0.3)
    by_head = [t.detach().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v)]  # [batch, heads, tokens, .] in memory
    turned = first.detach().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    for a, b in zip(attend(*by_head, turned, go.transpose(1, 2).contiguous().transpose(1, 2), last, g, 0.3), want):
        assert torch.equal(a, b)
    spread = [torch.zeros(2, 70, 4, 64, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    for s, t in zip(spread, (q, k, v)):
        s[..., ::2] = t.detach()
    for a, b in zip(attend(*(s[..., ::2].detach().requires_grad_() for s in spread), first, go, last, g, 0.3), want):
        assert torch.equal(a, b)
    one = k.detach()[:, :1].expand(2, 70, 4, 32)
    a, b = F.linear_attention(q, one, v, g), F.linear_attention(q, one.contiguous(), v, g)
    assert torch.equal(a, b)
    far = torch.empty(2**31 + 2**30 + 4096, dtype=torch.bfloat16, device=DEV)
    x = far.as_strided((1, 3, 4, 32), (0, (2**31 + 2**30) // 2, 64, 1))
    x.copy_(q.detach()[:1, :3])
    assert torch.equal(F.linear_attention(x, x, x, g), F.linear_attention(q[:1, :3], q[:1, :3], q[:1, :3], g))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_is_causal_for_values_that_are_not_finite(dtype):
    """An infinity or NaN of a token's key or value reaches that token and later ones, of its head, and, of a value, its column
    alone; one in a query its own row; in the gradients likewise backwards."""
    n, at = 100, 37
    g, scale = decays(5)[[0, 3, 4]], 0.3
    clean = inputs(5, (1, n), 3, 3, 32, 48, dtype, 1)
    want = attend(*clean, g, scale)
    for which, value in ((0, "nan"), (0, "inf"), (1, "nan"), (1, "inf"), (2, "nan"), (2, "-inf"), (4, "nan"), (4, "inf")):
        t = list(clean)
        bad = t[which].detach().clone()
        bad[0, at, 1, 7] = float(value)
        t[which] = bad.requires_grad_(which < 4)
        got = attend(*t, g, scale)
        hit = [torch.zeros_like(x, dtype=torch.bool) for x in want]  # out, state, gq, gk, gv, gs
        row, late, early = (0, at, 1), (0, slice(at, None), 1), (0, slice(None, at + 1), 1)
        if which == 0:  # q: its out; gk, gv of tokens up to it, gk in its column, gv and gs
            hit[0][row], hit[3][early], hit[4][early], hit[5][0, 1] = True, True, True, True
            hit[3][early] = False
            hit[3][0, :at + 1, 1, 7] = True
            hit[5][0, 1] = False
            hit[5][0, 1, 7] = True
        elif which == 1:  # k: out from it on, the state's row, gq's column from it on, gv's row
            hit[0][late], hit[1][0, 1, 7], hit[4][row] = True, True, True
            hit[2][0, at:, 1, 7] = True
        elif which == 2:  # v: out's column from it on, the state's column, gq from it on, gk's row
            hit[0][0, at:, 1, 7], hit[1][0, 1, :, 7], hit[3][row] = True, True, True
            hit[2][late] = True
        else:  # the gradient: gq's row, gk up to it, gv's column up to it, gs's column
            hit[2][row], hit[3][early], hit[4][0, :at + 1, 1, 7], hit[5][0, 1, :, 7] = True, True, True, True
        for name, a, b, h in zip(("out", "state", "gq", "gk", "gv", "gs"), got, want, hit):
            finite = torch.isfinite(a)
            assert not finite[h].any(), f"{which} {value} {name}: finite where it depends"
            assert torch.equal(a[~h], b[~h]), f"{which} {value} {name}: changed elsewhere"


def test_attention_missing_gradients():
    q, k, v, first, go, last = inputs(6, (2, 70), 4, 2, 32, 32, torch.float32, 2)
    g = decays(4)
    everything = torch.autograd.grad(F.linear_attention(q, k, v, g, first, final_state=True), [q, k, v, first], [go, last])
    out_only = torch.autograd.grad(F.linear_attention(q, k, v, g, first), [q, k, v, first], go)
    state_only = torch.autograd.grad(F.linear_attention(q, k, v, g, first, final_state=True)[1], [q, k, v, first], last, allow_unused=True)
    for a, b, c in zip(everything, out_only, state_only):
        assert (a - b - c).norm() <= 1e-6 * a.norm()
    assert not state_only[0].any()
    for i, t in enumerate((q, k, v, first)):
        args = [x if x is t else x.detach() for x in (q, k, v, first)]
        (one,) = torch.autograd.grad(F.linear_attention(args[0], args[1], args[2], g, args[3], final_state=True), [t], [go, last])
        assert torch.equal(one, everything[i])
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(F.linear_attention(q, k, v, g).sum(), q, create_graph=True)


def test_attention_repeats_itself():
    """The same results every time, whatever ran in between (no sums whose order changes)."""
    t = inputs(7, (2, 1500), 4, 2, 64, 64, torch.bfloat16, 2)
    g = decays(4)
    want = attend(*t, g, 0.2)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(attend(*t, g, 0.2), want))


# ------------------------------------------------------------------------------------------------
# A token at a time
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,dv", DIMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_step(dtype, dim, dv):
    """Steps in a cache, some of the batch without a place, against the oracle's whole sequence; other places stay."""
    heads, kvh, batch, cache = 4, 2, 5, 8
    g = decays(heads)
    state = randn(1, cache, heads, dim, dv)
    before = state.clone()
    slots = torch.tensor([6, -1, 0, 8, 3], dtype=torch.int32, device=DEV)
    rows = [[t[:, i] for t in inputs(10 * dim + dv, (batch, 3), heads, kvh, dim, dv, dtype, 0)[:3]] for i in range(3)]
    outs = []
    with torch.no_grad():
        for i, (q, k, v) in enumerate(rows):
            outs.append(F.linear_attention_step(q, k, v, g, state, slots.long() if i == 1 else slots, 0.3))
    out = torch.stack(outs, 1)
    q, k, v = (torch.stack([r[j] for r in rows], 1) for j in range(3))
    for b, slot in enumerate(slots.tolist()):
        if not 0 <= slot < cache:
            assert not out[b].any()
            continue
        check_sequence(dict(out=out[b], state=state[slot]), q[b], k[b], v[b], g, 0.3, before[slot], None, None, f"{b}")
    left = [i for i in range(cache) if i not in slots.tolist()]
    assert torch.equal(state[left], before[left])


@pytest.mark.parametrize("batch", [1, 3, 300, 1000])
def test_step_with_the_same_place_twice(batch):
    """Tokens of one place are taken one after another, wherever they stand in the batch."""
    heads, dim, cache = 2, 32, 4
    g = decays(heads)
    q, k, v, *_ = (t.detach() for t in inputs(3, (batch,), heads, 1, dim, dim, torch.float32, 0))
    slots = torch.randint(-1, cache, (batch,), generator=torch.Generator().manual_seed(1)).to(DEV)
    state = randn(1, cache, heads, dim, dim)
    before = state.clone()
    out = F.linear_attention_step(q, k, v, g, state, slots)
    for s in range(cache):
        rows = (slots == s).nonzero()[:, 0]
        check_sequence(dict(out=out[rows], state=state[s]), q[rows], k[rows], v[rows], g, dim**-0.5, before[s], None, None, f"{s}")
    assert not out[slots < 0].any()


def test_step_of_more_states_than_workgroups():
    batch, heads = 70000, 16
    q, k, v = randn(1, batch, heads, 2), randn(2, batch, heads, 2), randn(3, batch, heads, 1)
    state = randn(4, batch, heads, 2, 1)
    want = k.unsqueeze(-1) * v.unsqueeze(-2) + state  # one rounding apart: what is not lost is added as it is
    out = F.linear_attention_step(q, k, v, torch.zeros(heads, device=DEV), state, scale=1.0)
    size = k.abs().unsqueeze(-1) * v.abs().unsqueeze(-2) + 2 * want.abs()
    assert ((state - want).abs() <= 2.0**-22 * size).all()
    assert ((out.double() - (q.double().unsqueeze(-1) * state.double()).sum(-2)).abs() <= 2.0**-20 * (q.abs().unsqueeze(-1) * state.abs()).sum(-2)).all()


def test_step_strides_and_versions():
    heads, dim = 3, 32
    g = decays(heads)
    q, k, v, *_ = (t.detach() for t in inputs(4, (5,), heads, heads, dim, dim, torch.bfloat16, 0))
    plain = randn(1, 5, heads, dim, dim)
    layers = torch.stack([torch.zeros_like(plain), plain, torch.zeros_like(plain)], 2)  # [slots, heads, layers, dim, dim]
    by_head = plain.transpose(0, 1).contiguous().transpose(0, 1)
    want = F.linear_attention_step(q, k, v, g, plain)
    for state in (layers[:, :, 1], by_head):
        version = state._version
        assert torch.equal(F.linear_attention_step(q, k, v, g, state), want) and torch.equal(state, plain)
        assert state._version > version
    assert not layers[:, :, 0].any() and not layers[:, :, 2].any()
    wide = torch.stack([q, k, v], 2)
    state = randn(1, 5, heads, dim, dim)
    assert torch.equal(F.linear_attention_step(wide[:, :, 0], wide[:, :, 1], wide[:, :, 2], g, state), want)


def test_prompt_then_steps():
    """A packed prompt's last states go on token by token as the whole sequences would."""
    lengths, more, heads, kvh, dim, dv = [5, 0, 133, 64], 4, 4, 2, 64, 48
    g = decays(heads)
    offsets = torch.tensor([0, *np.cumsum(lengths)], device=DEV)
    whole = [[t.detach() for t in inputs(20 + i, (n + more,), heads, kvh, dim, dv, torch.bfloat16, 0)[:3]] for i, n in enumerate(lengths)]
    with torch.no_grad():
        q, k, v = (torch.cat([w[j][:n] for w, n in zip(whole, lengths)]) for j in range(3))
        out, last = F.linear_attention(q, k, v, g, offsets=offsets, final_state=True)
        cache = torch.zeros(6, heads, dim, dv, device=DEV)
        slots = torch.tensor([4, 1, 5, 0], device=DEV)
        cache[slots] = last
        steps = [F.linear_attention_step(*(torch.stack([w[j][n + i] for w, n in zip(whole, lengths)]) for j in range(3)), g, cache, slots) for i in range(more)]
    for i, (w, n) in enumerate(zip(whole, lengths)):
        got = torch.cat([out[offsets[i]:offsets[i + 1]], torch.stack([s[i] for s in steps])])
        check_sequence(dict(out=got, state=cache[slots[i]]), *w, g, dim**-0.5, None, None, None, f"{i}")


# ------------------------------------------------------------------------------------------------
# Together
# ------------------------------------------------------------------------------------------------


def block(x, w, p, f, g, heads, kvh, dim):
    """Projection, norm with rotation, attention: what a layer does."""
    joint = (x @ w).unflatten(-1, (heads + 2 * kvh, dim))
    q, k, v = joint.split([heads, kvh, kvh], -2)
    q, k = F.rms_norm_rotary(q, k, w.new_ones(dim), w.new_ones(dim), p, f)
    return F.linear_attention(q, k, v, g).flatten(-2)


def test_block_against_float64():
    """The operators one after another in float32 against the same formulas in float64, forward and gradients; the errors of three
    operators in turn, each below 2^-17 of its terms."""
    heads, kvh, dim, n = 4, 2, 32, 90
    x, w = randn(1, 2, n, 24).requires_grad_(), randn(2, 24, (heads + 2 * kvh) * dim, scale=0.2).requires_grad_()
    p, f, g, go = F.grid_positions([9, 10], device=DEV), F.rotary_frequencies([8, 8], device=DEV), decays(heads), randn(3, 2, n, heads * dim)
    y = block(x, w, p, f, g, heads, kvh, dim)
    got = [y, *torch.autograd.grad(y, [x, w], go)]

    x64, w64 = (t.detach().double().cpu().requires_grad_() for t in (x, w))
    joint = (x64 @ w64).unflatten(-1, (heads + 2 * kvh, dim))
    q, k, v = joint.split([heads, kvh, kvh], -2)
    angle = p.cpu().double() @ f.cpu()

    def turned(t):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
        a, b = t.chunk(2, -1)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    q, k, v = turned(q), turned(k).repeat_interleave(2, -2), v.repeat_interleave(2, -2)
    gap = torch.arange(n)[:, None] - torch.arange(n)
    weight = torch.where(gap == 0, 1.0, torch.where(gap > 0, torch.exp(g.cpu().double()[:, None, None] * gap.clamp_min(1)), 0.0))
    score = (q.transpose(1, 2) @ k.transpose(1, 2).transpose(-1, -2)) * weight * dim**-0.5
    y64 = (score @ v.transpose(1, 2)).transpose(1, 2).flatten(-2)
    want = [y64, *torch.autograd.grad(y64, [x64, w64], go.double().cpu())]
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).norm() <= 2.0**-15 * b.norm()


def test_captured_steps():
    """A training step of the block and a serving step in one graph each, every replay against the eager result."""
    heads, kvh, dim, n = 4, 2, 64, 300
    x, w = randn(1, 2, n, 32).requires_grad_(), randn(2, 32, (heads + 2 * kvh) * dim, scale=0.2).requires_grad_()
    p, f, g, go = torch.arange(n, device=DEV)[:, None], F.rotary_frequencies([32], device=DEV), decays(heads), randn(3, 2, n, heads * dim)
    tokens, cache, slots = randn(4, 3, heads + 2 * kvh, dim), randn(5, 6, heads, dim, dim), torch.tensor([5, -1, 2], device=DEV)

    def train():
        y = block(x, w, p, f, g, heads, kvh, dim)
        return [y, *torch.autograd.grad(y, [x, w], go)]

    def serve(state):
        with torch.no_grad():
            q, k, v = tokens.split([heads, kvh, kvh], -2)
            return [F.linear_attention_step(q, k, v, g, state, slots)]

    def warm(call):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        return graph, got

    graph, got = warm(train)
    steps, out = warm(lambda: serve(cache))
    for i in range(4):
        with torch.no_grad():
            x.copy_(randn(10 + i, 2, n, 32))
            tokens.copy_(randn(20 + i, *tokens.shape))
            cache.copy_(randn(30 + i, *cache.shape))
        other = cache.clone()
        graph.replay()
        steps.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, train()):
            assert torch.equal(a, b) or (a - b).norm() <= 1e-6 * b.norm(), f"replay {i}"
        assert torch.equal(out[0], serve(other)[0]) and torch.equal(cache, other), f"replay {i}"


def test_captured_packed_sequences():
    """Offsets are read on the device: a replay takes those that are there then."""
    heads, kvh, dim, dv, n = 2, 1, 32, 16, 1500
    q, k, v, first, go, last = inputs(9, (n,), heads, kvh, dim, dv, torch.bfloat16, 4)
    g = decays(heads)
    cuts = [[0, 0, 700, 1300, 1500], [3, 900, 900, 1100, 1499], [0, 1500, 1500, 1500, 1500], [500, 501, 502, 503, 504]]
    offsets = torch.tensor(cuts[0], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(q, k, v, first, go, last, g, 0.3, offsets)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attend(q, k, v, first, go, last, g, 0.3, offsets)
    for cut in cuts[1:] + cuts:
        offsets.copy_(torch.tensor(cut))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, attend(q, k, v, first, go, last, g, 0.3, offsets))), cut


def test_on_another_stream():
    t = inputs(8, (2, 700), 4, 2, 64, 64, torch.bfloat16, 2)
    g = decays(4)
    want = attend(*t, g, 0.2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(*t, g, 0.2)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
