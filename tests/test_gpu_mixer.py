"""The channel-mixing operators on the GPU against the float64 oracle (tests/mixer_oracle.py).

Tolerances, with u the unit roundoff of the output's type (2^-24, 2^-11, 2^-8) and f = 2^-24:
8-bit blocks are exact (codes and scales bit for bit). A norm's output is formed by a sum of C squares
(lane sums of at most 32 terms, then a tree of 10 levels: relative error below 45 f, halved by the root),
an addition, a root, a division and two products: 32 f relative, then the rounding to the output's type.
Gradients: 64 f of the sum of the terms' magnitudes, then the rounding. Sums over rows: 2 sqrt(rows) + 16
units f of the sum of magnitudes (the usual growth of a sum's rounding errors). The activation: 16 f
relative in float32 (exponential and division to 2 units each); in 16 bits the fast exponential adds |g| f.
Subnormal outputs add half their spacing.
"""
import numpy as np
import pytest
import torch

import morphocore_amd.functional as F
from tests import mixer_oracle as O

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


def near(got, want, size, dtype, what=""):
    """|got - want| <= size + u |want| + the subnormals' half spacing, elementwise."""
    got, far = np64(got), np.abs(np64(got) - want)
    assert got.shape == want.shape
    bad = far > size + U[dtype] * np.abs(want) + TINY[dtype]
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} values, first {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]}"


def same_packed(packed, x64, what=""):
    codes, scales = O.pack(x64)
    assert packed.codes.dtype == torch.float8_e4m3fn and packed.scales.dtype == torch.float8_e8m0fnu
    assert tuple(packed.codes.shape) == codes.shape and tuple(packed.scales.shape) == scales.shape
    assert np.array_equal(packed.scales.view(torch.uint8).cpu().numpy(), scales), what
    got = packed.codes.view(torch.uint8).cpu().numpy()
    nan = np.isnan(O.VALUES[codes])
    assert np.isnan(O.VALUES[got])[nan].all() and np.array_equal(got[~nan], codes[~nan]), what


# ------------------------------------------------------------------------------------------------
# 8-bit blocks
# ------------------------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 32), (3, 7), (2, 33), (5, 64), (4, 127), (2, 3, 100), (1, 2049), (70, 8), (7, 1000), (300, 31), (9000, 4)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
def test_pack_and_unpack(dtype, shape):
    x = randn(sum(shape), *shape, scale=3.0)
    x = (x * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=torch.Generator().manual_seed(1)).to(DEV))).to(dtype)
    packed = F.pack8(x)
    same_packed(packed, np64(x))
    want = O.unpack(packed.codes.view(torch.uint8).cpu().numpy(), packed.scales.view(torch.uint8).cpu().numpy())
    for to in (torch.float32, torch.bfloat16):
        got = F.unpack8(packed, to)
        assert got.dtype == to and np.array_equal(np64(got), want)
    with np.errstate(over="ignore"):
        half = np.clip(want, -65504, 65504).astype(np.float16).astype(np.float64)
    assert np.array_equal(np64(F.unpack8(packed, torch.float16)), half)


def test_pack_every_code_and_tie():
    """Every code's value, every midpoint of two codes, and their float32 neighbours, under several scales."""
    v = O.VALUES[:0x7F]
    mid = (v[:-1] + v[1:]) / 2
    pts = np.concatenate([v, mid, np.nextafter(mid.astype(np.float32), np.float32(np.inf)), np.nextafter(mid.astype(np.float32), np.float32(-np.inf))])
    pts = np.concatenate([pts, -pts]).astype(np.float32)
    pts = np.pad(pts, (0, -len(pts) % 31)).reshape(-1, 31)
    for e in (0, 5, -20, -117, 100, 119):
        x = np.concatenate([np.full((len(pts), 1), 448.0, np.float32), pts], axis=1) * np.float32(2.0) ** np.float32(e)
        same_packed(F.pack8(torch.from_numpy(x).to(DEV)), x.astype(np.float64), f"scale 2^{e}")


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_special_values(dtype):
    """Infinities and NaN in a block, the type's largest and smallest values, zeros of both signs."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(10, 64)
    x[0, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0])
    x[1, 5], x[1, 40] = big, -big
    x[2, 3], x[2, 4] = tiny, -tiny
    x[3, :] = float("nan")
    x[4, :] = -0.0
    x[5, 0], x[5, 1] = float("inf"), big
    x[6, ::7] = torch.finfo(dtype).min
    x[7, 33] = tiny / 4
    x[8, :] = torch.linspace(-1, 1, 64) * big
    x = x.to(dtype).to(DEV)
    packed = F.pack8(x)
    same_packed(packed, np64(x))
    got = F.unpack8(packed, torch.float32)
    assert torch.isfinite(got[4:5]).all() and torch.isfinite(got[8]).all() and torch.isnan(got[3]).all()
    if dtype == torch.float16:
        assert torch.isfinite(F.unpack8(packed, dtype)[8]).all()


def test_pack_reads_strided_rows_and_other_orders():
    wide = randn(3, 6, 5, 200)
    for x in (wide[..., 40:140], wide[:, 2, 1:98], wide.transpose(0, 1), wide.transpose(1, 2), wide[:, :, ::2], wide[::2], wide[:1].expand(4, 5, 200),
              wide[0, 0, :1].expand(3, 40), wide[0, 0], wide[:, :, :1]):
        a, b = F.pack8(x), F.pack8(x.contiguous())
        assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))
        assert a.codes.shape == x.shape


@pytest.mark.parametrize("shape", [(0, 5), (3, 0), (0,), (2, 0, 7)])
def test_empty(shape):
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    p = F.pack8(x)
    assert p.codes.shape == x.shape and F.unpack8(p).shape == x.shape
    w = torch.ones(shape[-1], device=DEV, requires_grad=True)
    y, packed, h = F.rms_norm8(x, w, torch.zeros_like(x))
    gx, gw = torch.autograd.grad([y, h], [x, w], [torch.ones_like(y), torch.ones_like(h)])
    assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w)) and packed.codes.shape == x.shape
    both = torch.zeros(shape[:-1] + (2 * shape[-1],), device=DEV, requires_grad=True)
    y, packed = F.gated_silu8(both)
    assert y.shape == x.shape and torch.autograd.grad(y, both, torch.zeros_like(y))[0].shape == both.shape
    gy = torch.zeros(shape[:-1] + (3,), device=DEV)
    assert torch.equal(F.grad_weight8(gy, p), torch.zeros(3, shape[-1], device=DEV))


# ------------------------------------------------------------------------------------------------
# Root-mean-square norm
# ------------------------------------------------------------------------------------------------

NORMS = [(1, 1), (3, 5), (2, 32), (17, 33), (130, 64), (9, 120), (33, 250), (7, 500), (5, 777), (6, 1024), (3, 1237), (4, 2048), (3, 2500), (2, 4096),
         (2, 5001), (3, 8192), (2, 11000), (2, 12289), (1, 20000), (2, 32801), (2100, 40), (700, 130)]


def check_norm(dtype, wdtype, rows, cols, residual, gy_on=True, gh_on=True, scale=1.0):
    x = randn(rows * 7 + cols, rows, cols, dtype=dtype, scale=scale).requires_grad_()
    w = (1 + 0.2 * randn(cols, cols)).to(wdtype).requires_grad_()
    r = randn(rows + cols * 3, rows, cols, dtype=dtype, scale=scale).requires_grad_() if residual else None
    eps = 1e-5
    y, packed, h = F.rms_norm8(x, w, r, eps)
    assert y.dtype == dtype
    sum64 = np64(x) + np64(r) if residual else np64(x)
    want = O.rms_norm(sum64, np64(w), eps)
    near(y, want, 32 * f32 * np.abs(want), dtype, "y")
    same_packed(packed, np64(y))
    if residual:
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
        plain = F.rms_norm(x, w, r, eps)
        assert torch.equal(plain[0], y) and torch.equal(plain[1], h)
    else:
        assert h is None and torch.equal(F.rms_norm(x, w, eps=eps), y)
    with torch.no_grad():
        alone = F.rms_norm8(x, w, r, eps, full=False)
        assert alone.y is None and torch.equal(alone.packed.codes.view(torch.uint8), packed.codes.view(torch.uint8))
    gy, gh = randn(5, rows, cols, dtype=dtype, scale=0.1), randn(6, rows, cols, dtype=dtype, scale=0.1)
    outs = [(y, gy)] * gy_on + [(h, gh)] * (gh_on and residual)
    leaves = [x, w] + [r] * residual
    grads = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs], allow_unused=True)
    # The stored h, with the forward's rstd: of the unrounded sum.
    h64 = np64(h) if residual else np64(x)
    rstd = 1 / np.sqrt(np.mean(sum64**2, axis=-1, keepdims=True) + eps)
    n, a = h64 * rstd, (np64(gy) if gy_on else 0 * h64) * np64(w)
    m, gh64 = np.mean(a * n, axis=-1, keepdims=True), np64(gh) if gh_on and residual else 0.0
    gx = rstd * (a - n * m) + gh64
    size = rstd * (np.abs(a) + np.abs(n) * np.mean(np.abs(a * n), axis=-1, keepdims=True)) + np.abs(gh64)
    near(grads[0], gx, 64 * f32 * size, dtype, "gx")
    terms = np64(gy) * n if gy_on else 0 * n
    near(grads[1], terms.sum(0), (2 * np.sqrt(rows) + 16) * f32 * np.abs(terms).sum(0), wdtype, "gw")
    if residual:
        assert torch.equal(grads[2], grads[0])


@pytest.mark.parametrize("rows,cols", NORMS)
@pytest.mark.parametrize("dtype", TYPES)
def test_norm(dtype, rows, cols):
    check_norm(dtype, dtype, rows, cols, residual=True)
    check_norm(dtype, torch.float32, rows, cols, residual=False)


@pytest.mark.parametrize("cols", [64, 500, 4096, 33000])
def test_norm_with_one_gradient_missing(cols):
    check_norm(torch.bfloat16, torch.bfloat16, 5, cols, True, gy_on=False)
    check_norm(torch.float32, torch.float32, 5, cols, True, gh_on=False)


def test_only_the_gradients_asked_for():
    x, r, w = randn(1, 9, 200).requires_grad_(), randn(2, 9, 200).requires_grad_(), randn(3, 200).requires_grad_()
    gy, gh = randn(4, 9, 200), randn(5, 9, 200)
    def grads(a, b, c):
        return torch.autograd.grad(F.rms_norm(a, b, c), [t for t in (a, b, c) if t.requires_grad], [gy, gh])
    gx, gw, gr = grads(x, w, r)
    assert torch.equal(grads(x, w.detach(), r.detach())[0], gx) and torch.equal(grads(x.detach(), w.detach(), r)[0], gr)
    assert torch.equal(grads(x.detach(), w, r.detach())[0], gw)
    u = randn(6, 9, 200).requires_grad_()
    for f in (F.gated_silu, lambda *t: F.gated_silu8(*t).y):
        gg, gu = torch.autograd.grad(f(x, u), [x, u], gy)
        assert torch.equal(torch.autograd.grad(f(x, u.detach()), x, gy)[0], gg)
        assert torch.equal(torch.autograd.grad(f(x.detach(), u), u, gy)[0], gu)


def test_norm_of_expanded_and_strided_rows():
    base = randn(1, 4, 6, 300).requires_grad_()
    w = randn(2, 100).requires_grad_()
    gy = randn(3, 4, 6, 100)
    for view in (lambda t: t[..., 50:150], lambda t: t[..., 1:300:3][..., :100], lambda t: t[:1, :, :100].expand(4, 6, 100),
                 lambda t: t.transpose(0, 1)[..., :100].transpose(0, 1)):
        got = torch.autograd.grad(F.rms_norm(view(base), w), [base, w], gy)
        want = torch.autograd.grad(F.rms_norm(view(base).contiguous(), w), [base, w], gy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # A gradient that is an expanded value, as sum() gives.
    x = randn(4, 5, 64).requires_grad_()
    a, = torch.autograd.grad(F.rms_norm(x, w[:64]).sum(), x)
    b, = torch.autograd.grad(F.rms_norm(x, w[:64]), x, torch.ones(5, 64, device=DEV))
    assert torch.equal(a, b)


def test_norm_gradient_is_the_forwards_difference():
    x, w, gy = randn(1, 3, 200).requires_grad_(), (1 + 0.1 * randn(2, 200)).requires_grad_(), randn(3, 3, 200)
    gx, gw = torch.autograd.grad(F.rms_norm(x, w), [x, w], gy)
    d, dw, t = randn(4, 3, 200), randn(5, 200), 2.0**-7
    def loss(a, b):
        return (F.rms_norm(a, b).double() * gy).sum().item()
    with torch.no_grad():
        # Second-order differences: truncation t^2 of the third derivative, rounding f / t of the loss's terms.
        size = (gx.abs() * d.abs()).sum().item()
        assert abs((loss(x + t * d, w) - loss(x - t * d, w)) / (2 * t) - (gx * d).sum().item()) <= 2e-3 * size
        size = (gw.abs() * dw.abs()).sum().item()
        assert abs((loss(x, w + t * dw) - loss(x, w - t * dw)) / (2 * t) - (gw * dw).sum().item()) <= 1e-3 * size


def test_norm_special_rows():
    """A zero row, a row with an infinity, a row with a NaN, a row of the type's lowest value: each by itself."""
    x = randn(1, 6, 96)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    x[4] = torch.finfo(torch.float32).min
    w = torch.ones(96, device=DEV)
    y, packed, _ = F.rms_norm8(x, w)
    want = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.allclose(y[ok], want[ok], rtol=1e-5, atol=1e-6)
    same_packed(packed, np64(y))


# ------------------------------------------------------------------------------------------------
# Gated activation
# ------------------------------------------------------------------------------------------------

def check_gated(dtype, rows, cols, joint, scale=2.0):
    x = randn(rows + cols, rows, 2 * cols, dtype=dtype, scale=scale)
    if joint:
        leaves = [x.requires_grad_()]
        args = (x,)
    else:
        leaves = [x[:, :cols].clone().requires_grad_(), x[:, cols:].clone().requires_grad_()]
        args = tuple(leaves)
    g, u = np64(x)[:, :cols], np64(x)[:, cols:]
    fast = 0.0 if dtype == torch.float32 else f32
    want = O.gated(g, u)
    y, packed = F.gated_silu8(*args)
    near(y, want, (16 * f32 + fast * np.abs(g)) * np.abs(want), dtype, "y")
    same_packed(packed, np64(y))
    plain = F.gated_silu(*args)
    assert torch.equal(plain, y)
    gy = randn(9, rows, cols, dtype=dtype, scale=0.1)
    for out, gk, uk in ((plain, g, u), (y, O.unpack(*O.pack(g)), O.unpack(*O.pack(u)))):
        got = torch.autograd.grad(out, leaves, gy)
        got = [got[0][:, :cols], got[0][:, cols:]] if joint else got
        gg, gu, size = O.gated_grads(gk, uk, np64(gy))
        near(got[0], gg, (16 * f32 + fast * np.abs(gk)) * size, dtype, "grad gate")
        near(got[1], gu, (16 * f32 + fast * np.abs(gk)) * np.abs(gu), dtype, "grad up")


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 31), (3, 32), (5, 100), (64, 256), (7, 1021), (3, 2048), (2, 2731), (70000, 8)])
@pytest.mark.parametrize("joint", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated(dtype, joint, rows, cols):
    check_gated(dtype, rows, cols, joint)


def test_gated_far_values():
    """Gates from -200 to 200: the exponential overflows and underflows without a NaN."""
    g = torch.linspace(-200, 200, 4001, device=DEV).view(1, -1).requires_grad_()
    u = torch.full_like(g, 1.5).requires_grad_()
    y = F.gated_silu(g, u)
    gg, gu = torch.autograd.grad(y, [g, u], torch.ones_like(y))
    want = O.gated(np64(g), np64(u))
    wg, wu, size = O.gated_grads(np64(g), np64(u), np.ones(1))
    # exp(-g) beyond float32 leaves 0 for values below 2^-126.
    near(y, want, 16 * f32 * np.abs(want) + 2.0**-118, torch.float32)
    near(gg, wg, 16 * f32 * size + 2.0**-118, torch.float32)
    near(gu, wu, 16 * f32 * np.abs(wu) + 2.0**-118, torch.float32)


def test_gated_slices():
    x = randn(1, 3, 4, 500, dtype=torch.bfloat16).requires_grad_()
    a, b = x[..., 10:210], x[..., 250:450]
    gy = randn(2, 3, 4, 200, dtype=torch.bfloat16)
    for f in (lambda *t: F.gated_silu(*t), lambda *t: F.gated_silu8(*t).y):
        got, = torch.autograd.grad(f(a, b), x, gy)
        want, = torch.autograd.grad(f(a.contiguous(), b.contiguous()), x, gy)
        joint, = torch.autograd.grad(f(torch.cat([a, b], -1)), x, gy)
        assert torch.equal(got, want) and torch.equal(got, joint)


# ------------------------------------------------------------------------------------------------
# Weight gradient
# ------------------------------------------------------------------------------------------------

WEIGHTS = [(1, 1, 1), (1, 64, 64), (31, 5, 33), (32, 64, 32), (100, 64, 64), (257, 100, 31), (300, 33, 257), (511, 129, 130), (1000, 256, 300),
           (5003, 70, 65), (8200, 1000, 1030), (33000, 300, 500), (4096, 128, 512), (777, 513, 40), (64, 300, 1000), (20000, 16, 24), (300, 9, 301), (300, 301, 9), (50, 8, 8), (70, 7, 200), (70, 200, 7), (9, 200, 250)]


@pytest.mark.parametrize("rows,out,cols", WEIGHTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_weight_gradient(dtype, rows, out, cols):
    packed = F.pack8(randn(rows + cols, rows, cols) * torch.exp(randn(3, rows, 1)))
    gy = randn(rows + out, rows, out, dtype=dtype, scale=0.1)
    x64 = O.unpack(packed.codes.view(torch.uint8).cpu().numpy(), packed.scales.view(torch.uint8).cpu().numpy())
    g64 = np64(gy)
    want, size = g64.T @ x64, np.abs(g64).T @ np.abs(x64)
    for to in (None, torch.float32):
        got = F.grad_weight8(gy, packed, to)
        assert got.dtype == (to or dtype)
        near(got, want, (2 * np.sqrt(rows) + 16) * f32 * size, got.dtype, f"dtype {to}")


# Outputs large enough for the wide and the tall tiles, unsplit and split, with edges inside a tile.
@pytest.mark.parametrize("rows,out,cols", [(333, 4050, 4060), (290, 4060, 2030), (4100, 1020, 2040), (17, 2050, 4100)])
@pytest.mark.parametrize("dtype", TYPES)
def test_weight_gradient_of_large_outputs(dtype, rows, out, cols):
    test_weight_gradient(dtype, rows, out, cols)


@pytest.mark.parametrize("dtype", TYPES)
def test_weight_gradient_keeps_every_bit_of_its_operands(dtype):
    """One row: the products alone, each exact but for the last rounding."""
    gy = randn(1, 1, 70, dtype=dtype) * torch.exp2(torch.arange(70, device=DEV) % 9 - 4.0).to(dtype)
    packed = F.pack8(randn(2, 1, 90) * 100)
    x64 = O.unpack(packed.codes.view(torch.uint8).cpu().numpy(), packed.scales.view(torch.uint8).cpu().numpy())
    want = (np64(gy).T @ x64).astype(np.float32)
    assert np.array_equal(F.grad_weight8(gy, packed, torch.float32).cpu().numpy(), want)


def test_weight_gradient_of_subnormal_values():
    """bfloat16 and float16 gradients down to their smallest values, float32 ones to 2^-133."""
    packed = F.pack8(torch.full((1, 40), 2.0**60, device=DEV))
    for dtype, e in ((torch.bfloat16, -131), (torch.float16, -22), (torch.float32, -109), (torch.float32, -124)):
        gy = (1 + torch.rand(1, 50, generator=torch.Generator().manual_seed(1), dtype=torch.float64)).mul(2.0**e).to(dtype).to(DEV)
        far = np.abs(np64(F.grad_weight8(gy, packed, torch.float32)) / 2.0**60 - np64(gy).T)
        assert far.max() <= (2.0**-133 if e == -124 else 0.0)


def test_weight_gradient_of_strided_and_expanded_gradients():
    packed = F.pack8(randn(1, 4, 50, 96))
    wide = randn(2, 4, 50, 200)
    for gy in (wide[..., 7:107], wide.transpose(0, 1)[:, :, :100].transpose(0, 1), wide[:1, :1, :100].expand(4, 50, 100), wide[..., ::2]):
        assert torch.equal(F.grad_weight8(gy, packed), F.grad_weight8(gy.contiguous(), packed))


def test_weight_gradient_is_the_same_every_time():
    packed, gy = F.pack8(randn(1, 30000, 64)), randn(2, 30000, 64)
    first = F.grad_weight8(gy, packed)
    assert all(torch.equal(F.grad_weight8(gy, packed), first) for _ in range(5))


def test_weight_gradient_not_finite():
    """An infinity or NaN reaches its own row or column of the gradient only."""
    for dtype in TYPES:
        gy, x = randn(1, 40, 70, dtype=dtype), randn(2, 40, 80)
        gy[3, 5], gy[4, 6], x[7, 9] = float("inf"), float("nan"), float("inf")
        got = F.grad_weight8(gy, F.pack8(x))
        bad = ~torch.isfinite(got)
        want = torch.zeros_like(bad)
        want[5], want[6], want[:, 9] = True, True, True
        assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear8_of_strides_without_a_matrix_view(dtype):
    """Exchanged leading dimensions, expanded gradients and a transposed weight: the products of the dense tensors, bit for bit."""
    x, w = randn(1, 20, 6, 64, dtype=dtype).transpose(0, 1), randn(2, 64, 40, dtype=dtype, scale=0.1).t()
    assert torch.equal(F.linear8(x, w), F.linear8(x.contiguous(), w))
    gy = randn(3, 20, 6, 40, dtype=dtype).transpose(0, 1)
    for g in (gy, gy[:, :1].expand(6, 20, 40)):
        got, want = [], []
        for a, b, out in ((x, g, got), (x.contiguous(), g.contiguous(), want)):
            a, v = a.detach().requires_grad_(), w.detach().requires_grad_()
            y = F.linear8(a, v)
            y += 1  # the output is no view
            out += [y, *torch.autograd.grad(y, [a, v], b), *torch.autograd.grad(F.linear8(a, w), a, b)]
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    near(F.linear8(x, w), np64(x) @ np64(w).T, 64 * f32 * (np.abs(np64(x)) @ np.abs(np64(w)).T), dtype)
    assert F.linear8(x[0, 0], w).shape == (40,) and F.linear8(x[:0], w).shape == (0, 20, 40) and F.linear8(x[..., :0], w[:, :0]).shape == (6, 20, 40)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear8(dtype):
    x, w = randn(1, 3, 20, 96, dtype=dtype).requires_grad_(), randn(2, 50, 96, dtype=dtype, scale=0.1).requires_grad_()
    gy = randn(3, 3, 20, 50, dtype=dtype)
    y = F.linear8(x, w)
    assert torch.equal(y, torch.nn.functional.linear(x, w))
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    packed = F.pack8(x)
    assert torch.equal(gw, F.grad_weight8(gy, packed))
    assert torch.equal(gx, gy @ w)
    gw2, = torch.autograd.grad(F.linear8(x, w, packed), w, gy)
    assert torch.equal(gw2, gw)
    # Only what is asked for is kept.
    assert torch.equal(torch.autograd.grad(F.linear8(x.detach(), w), w, gy)[0], gw)
    assert torch.equal(torch.autograd.grad(F.linear8(x, w.detach()), x, gy)[0], gx)


# ------------------------------------------------------------------------------------------------
# Streams, graphs, refusals that need a device
# ------------------------------------------------------------------------------------------------

def test_on_another_stream_and_in_a_graph():
    x, r, w = randn(1, 64, 256), randn(2, 64, 256), 1 + 0.1 * randn(3, 256)
    gy, up = randn(4, 64, 128), randn(5, 128, 256)

    def step():
        y, packed, h = F.rms_norm8(x, w, r)
        z, packed2 = F.gated_silu8(y)
        return [y, h, z, F.unpack8(packed), F.unpack8(packed2), F.grad_weight8(gy, packed), F.grad_weight8(y, packed2)]

    with torch.no_grad():
        want = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for i in range(4):
            x.copy_(randn(10 + i, 64, 256))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, step())), f"replay {i}"


def test_refusals_on_the_device():
    x, w = randn(1, 4, 64).requires_grad_(), randn(2, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="full=False"):
        F.rms_norm8(x, w, full=False)
    y = F.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="expected scalar type"):
        F.rms_norm(x, w.half())
    with pytest.raises(RuntimeError, match="expects every tensor on"):
        F.rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        F.pack8(x.double())
    with pytest.raises(RuntimeError, match="not implemented for 'Int'"):
        F.gated_silu(torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="expected scalar type"):
        F.linear8(x, randn(1, 5, 64).half())
    p = F.pack8(x)
    with pytest.raises(RuntimeError, match="dtype must be"):
        F.grad_weight8(randn(1, 4, 8), p, torch.float16)


def test_checkpoint8():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(96, 64), torch.nn.Dropout(0.5), torch.nn.Tanh()).to(DEV)
    x, gy = randn(1, 8, 96).requires_grad_(), randn(2, 8, 64)
    torch.manual_seed(7)
    out = F.checkpoint8(net, x)
    after = torch.rand(3, device=DEV)
    got = torch.autograd.grad(out, [x, *net.parameters()], gy)
    torch.manual_seed(7)
    kept = F.unpack8(F.pack8(x)).requires_grad_()
    assert torch.equal(net(x), out) and torch.equal(torch.rand(3, device=DEV), after)
    torch.manual_seed(7)
    want = torch.autograd.grad(net(kept), [kept, *net.parameters()], gy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        torch.manual_seed(7)
        assert torch.equal(F.checkpoint8(net, x), out)
    # Frozen parameters and an input without a gradient.
    net[0].weight.requires_grad_(False)
    net.eval()
    gb, = torch.autograd.grad(F.checkpoint8(net, x.detach()), net[0].bias, gy)
    assert torch.equal(gb, torch.autograd.grad(net(F.unpack8(F.pack8(x))), net[0].bias, gy)[0])


def test_autocast():
    """Operators keep their operands' type under autocast; a checkpointed module runs again under the forward's."""
    import morphocore_amd.nn as nn

    x, w = randn(1, 8, 96).requires_grad_(), randn(2, 40, 96).requires_grad_()
    mixer, net = nn.ChannelMixer(96, 64).to(DEV), torch.nn.Linear(96, 33).to(DEV)
    want = mixer(x)[0]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert F.linear8(x, w).dtype == torch.float32
        assert torch.equal(mixer(x)[0], want)
        out = F.checkpoint8(net, x)
    assert out.dtype == torch.bfloat16
    kept = F.unpack8(F.pack8(x)).requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        plain = net(kept)
    gy = randn(3, 8, 33, dtype=torch.bfloat16)
    for a, b in zip(torch.autograd.grad(out, [x, net.weight], gy), torch.autograd.grad(plain, [kept, net.weight], gy)):
        assert torch.equal(a, b)


def test_checkpoint8_of_modules_that_pass_or_drop_their_input():
    x = randn(1, 4, 32).requires_grad_()
    assert torch.equal(torch.autograd.grad(F.checkpoint8(torch.nn.Identity(), x), x, x.detach())[0], x)

    class Constant(torch.nn.Module):
        def forward(self, t):
            return torch.ones_like(t)

    out = F.checkpoint8(Constant(), x)
    assert torch.autograd.grad(out, x, x.detach(), allow_unused=True)[0] is None


# ------------------------------------------------------------------------------------------------
# Modules
# ------------------------------------------------------------------------------------------------

def test_channel_mixer_against_float64():
    """Outputs as a float64 block's; gradients within 1/16 of it by norm, the most that a kept value may be off."""
    import copy

    import morphocore_amd.nn as nn

    torch.manual_seed(0)
    m = nn.ChannelMixer(96, 160).to(DEV)
    x, r = randn(1, 2, 30, 96).requires_grad_(), randn(2, 2, 30, 96).requires_grad_()
    go, gh = randn(3, 2, 30, 96), randn(4, 2, 30, 96)
    out, h = m(x, r)
    got = torch.autograd.grad([out, h], [x, r, *m.parameters()], [go, gh])
    d = copy.deepcopy(m).double()
    xd, rd = x.detach().double().requires_grad_(), r.detach().double().requires_grad_()
    hd = xd + rd
    y = hd * torch.rsqrt(hd.square().mean(-1, keepdim=True) + 1e-6) * d.norm.weight
    g, u = (y @ d.expand.t()).chunk(2, -1)
    od = (g * torch.sigmoid(g) * u) @ d.contract.t()
    want = torch.autograd.grad([od, hd], [xd, rd, *d.parameters()], [go.double(), gh.double()])
    assert (out.double() - od).norm() <= 1e-5 * od.norm() and (h.double() - hd).norm() <= 1e-6 * hd.norm()
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= b.norm() / 16
    # Channels of images, as the morphological layers hold them.
    first = nn.ChannelMixer(96, 160, channels_first=True).to(DEV)
    first.load_state_dict(m.state_dict())
    xi = randn(5, 2, 96, 6, 7)
    out, h = first(xi)
    last, _ = m(xi.permute(0, 2, 3, 1))
    assert torch.equal(h, xi) and torch.equal(out, last.permute(0, 3, 1, 2))


def test_checkpoint8_of_a_morphological_stack():
    import morphocore_amd.nn as nn

    torch.manual_seed(0)
    stack = nn.MorphoStack(nn.Dilation(3, 4, 3, "max"), nn.SMorph(4, 4, 3, "sum", init_alpha=2.0), nn.Erosion(4, 3, 3, "min")).to(DEV)
    with torch.no_grad():
        for p in stack.parameters():
            p.add_(0.1 * torch.randn_like(p))
    x, gy = torch.rand(2, 3, 20, 33, device=DEV).requires_grad_(), randn(1, 2, 3, 20, 33)
    out = nn.Checkpoint8(stack)(x)
    assert torch.equal(out, stack(x))
    got = torch.autograd.grad(out, [x, *stack.parameters()], gy)
    kept = F.unpack8(F.pack8(x)).requires_grad_()
    want = torch.autograd.grad(stack(kept), [kept, *stack.parameters()], gy)
    # The stack's own gradient sums may differ in their order from run to run.
    assert all((a - b).norm() <= 1e-5 * b.norm() for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------
# Launches beyond the last-level cache, offsets past 32 bits
# ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,rows,cols", [(torch.bfloat16, 41000, 1001), (torch.float32, 300000, 88), (torch.float16, 2500, 17000)])
def test_large_launches_give_the_rows_of_small_ones(dtype, rows, cols):
    """More than 256 MB, whose results are stored past the caches: every row as the same row of a short array."""
    x, r = randn(1, 1000, cols, dtype=dtype).repeat(rows // 1000 + 1, 1)[:rows], randn(2, 1000, cols, dtype=dtype).repeat(rows // 1000 + 1, 1)[:rows]
    w = (1 + 0.1 * randn(3, cols)).to(dtype)

    def step(x, r):
        x, r = x.clone().requires_grad_(), r.clone().requires_grad_()
        y, packed, h = F.rms_norm8(x, w, r)
        gx, = torch.autograd.grad([y, h], x, [r.detach(), x.detach()])
        z, packed2 = F.gated_silu8(x, r)
        g, u = torch.autograd.grad(z, [x, r], y.detach())
        return [y, h, F.unpack8(packed, dtype), gx, z, F.unpack8(packed2, dtype), g, u]

    for large, small in zip(step(x, r), step(x[:1000], r[:1000])):
        assert torch.equal(large[:1000], small) and torch.equal(large[-500:], small[torch.arange(rows - 500, rows, device=DEV) % 1000])


def test_rows_past_32_bit_offsets():
    """Arrays of more than 2^32 elements: the last rows are worked on as the same rows of a small array."""
    rows, cols, tail = (1 << 26) + 5, 72, 300
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-tail:] = randn(1, tail, cols, dtype=torch.bfloat16)
    small = x[-tail:].clone()
    print("pack8 / unpack8", flush=True)
    p, q = F.pack8(x), F.pack8(small)
    assert torch.equal(p.codes[-tail:].view(torch.uint8), q.codes.view(torch.uint8))
    assert torch.equal(p.scales[-tail:].view(torch.uint8), q.scales.view(torch.uint8))
    assert torch.equal(F.unpack8(p, torch.bfloat16)[-tail:], F.unpack8(q, torch.bfloat16))
    print("grad_weight8", flush=True)
    # All other rows are zeros, so the sums are the small array's; the order differs.
    g64, x64 = np64(small[:, :64]), O.unpack(q.codes.view(torch.uint8).cpu().numpy(), q.scales.view(torch.uint8).cpu().numpy())
    got = F.grad_weight8(x[:, :64], p, torch.float32)
    near(got, g64.T @ x64, (2 * np.sqrt(tail) + 16) * f32 * (np.abs(g64).T @ np.abs(x64)), torch.float32, "gw")
    print("gated", flush=True)
    assert torch.equal(F.gated_silu(x)[-tail:], F.gated_silu(small))
    del p
    print("rms_norm", flush=True)
    w = torch.ones(cols, dtype=torch.bfloat16, device=DEV)
    assert torch.equal(F.rms_norm(x, w)[-tail:], F.rms_norm(small, w))
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_trains(dtype):
    """The example's network, through every operator: its loss falls to less than half."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_mixer.py")
    spec = importlib.util.spec_from_file_location("train_mixer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, kept = example.train(steps=40, size=32, batch=2, channels=16, dtype=dtype)
    assert all(np.isfinite(losses)) and kept > 0
    assert np.mean(losses[-5:]) < 0.5 * losses[0]
