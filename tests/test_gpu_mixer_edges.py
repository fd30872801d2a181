"""The channel-mixing operators on the GPU where their results are easily lost: checkpoints of modules that draw
numbers, write to their input or run under autocast, captured steps, empty tensors, missing gradients, values that
are not finite, the norm's gradients against the sum that its forward took, its widest rows."""
import numpy as np
import pytest
import torch

import morphocore_amd.functional as F
import morphocore_amd.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda"


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


class Noise(torch.nn.Module):
    """Draws whatever its training flag."""

    def forward(self, x):
        return x * torch.rand_like(x)


def test_checkpoint_draws_the_forwards_numbers():
    """A container in evaluation with a part in training, and a module that draws in evaluation too."""
    torch.manual_seed(0)
    mixed = torch.nn.Sequential(torch.nn.Linear(64, 48), torch.nn.Dropout(0.5)).to(DEV).eval()
    mixed[1].train()
    noise = torch.nn.Sequential(torch.nn.Linear(64, 48), Noise()).to(DEV).eval()
    x, gy = F.unpack8(F.pack8(randn(1, 9, 64))), randn(2, 9, 48)  # values that a checkpoint holds exactly
    for net in (mixed, noise):
        results = []
        for call in (net, lambda t: F.checkpoint8(net, t)):
            torch.manual_seed(7)
            a = x.clone().requires_grad_()
            out = call(a)
            results.append([out, *torch.autograd.grad(out, [a, *net.parameters()], gy), torch.rand(3, device=DEV)])
        for plain, kept in zip(*results):
            assert torch.equal(plain, kept)


def test_captured_step_of_a_checkpoint():
    """Forward and backward of checkpointed morphological layers and a channel mixer in one graph, whose every replay gives the eager
    step's results; with the generators' states to keep, the capture is refused."""
    torch.manual_seed(0)
    net = nn.Checkpoint8(torch.nn.Sequential(nn.Opening(8, 8, 3), nn.Closing(8, 8, 3)), preserve_rng=False).to(DEV)
    mixer = nn.ChannelMixer(8, 16, channels_first=True).to(DEV)
    with torch.no_grad():
        for p in net.parameters():
            p.add_(0.1 * torch.randn_like(p))
    params = [*net.parameters(), *mixer.parameters()]
    x, go = randn(1, 2, 8, 20, 33).requires_grad_(), randn(2, 2, 8, 20, 33)

    def step():
        out, h = mixer(net(x), x)
        return [out, h, *torch.autograd.grad([out, h], [x, *params], [go, go])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(randn(10 + i, 2, 8, 20, 33))
        graph.replay()
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(got, step())):
            assert torch.equal(a, b) or (a - b).norm() <= 1e-5 * b.norm(), f"replay {i}, result {k}"
    net.preserve_rng = True
    with pytest.raises(RuntimeError, match="preserve_rng=False"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            net(x)


def test_checkpoint_leaves_no_cast_weights_behind():
    """Under autocast: the gradients of a backward inside the region, and those of a weight that the same region uses again without the
    checkpoint."""
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(96, 96), torch.nn.Tanh()).to(DEV)
    x, gy = F.unpack8(F.pack8(randn(1, 8, 96))), randn(2, 8, 96, dtype=torch.bfloat16)

    def step(call, inside):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = call(x) + net(x)
            if inside:
                return [out, *torch.autograd.grad(out, net.parameters(), gy)]
        return [out, *torch.autograd.grad(out, net.parameters(), gy)]

    want = step(net, False)
    for inside in (False, True):
        for a, b in zip(step(lambda t: F.checkpoint8(net, t), inside), want):
            assert (a - b).norm() <= 2.0**-7 * b.norm()  # the two uses' bfloat16 gradients are added in another order
    with torch.autocast("cuda", dtype=torch.bfloat16):
        alone = torch.autograd.grad(F.checkpoint8(net, x), net.parameters(), gy)
        plain = torch.autograd.grad(net(x), net.parameters(), gy)
    assert all(torch.equal(a, b) for a, b in zip(alone, plain))


def test_gradients_inside_an_autocast_region():
    """linear8 and ChannelMixer keep their operands' type in a backward that runs inside the region: bit for bit the gradients outside."""
    torch.manual_seed(0)
    x, w, gy = randn(1, 8, 96).requires_grad_(), randn(2, 40, 96).requires_grad_(), randn(3, 8, 40)
    mixer, go = nn.ChannelMixer(96, 64).to(DEV), randn(4, 8, 96)

    def step():
        out, h = mixer(x)
        return [*torch.autograd.grad(F.linear8(x, w), [x, w], gy), *torch.autograd.grad([out, h], [x, *mixer.parameters()], [go, go])]

    want = step()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.parametrize("rows,cols", [((0,), 8), ((2, 0), 5), ((3,), 0), ((0,), 0), ((), 0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_empty_steps(dtype, rows, cols):
    """Forward and backward of every operator without rows or without columns."""
    def empty(n):
        return torch.zeros(*rows, n, dtype=dtype, device=DEV, requires_grad=True)

    joint, gate, up, w = empty(2 * cols), empty(cols), empty(cols), torch.ones(cols, dtype=dtype, device=DEV, requires_grad=True)
    for y, leaves in ((F.gated_silu(joint), [joint]), (F.gated_silu(gate, up), [gate, up]), (F.gated_silu8(joint).y, [joint]),
                      (F.gated_silu8(gate, up).y, [gate, up]), (F.rms_norm(gate, w), [gate, w]), (F.rms_norm(gate, w, up)[0], [gate, w, up]),
                      (F.rms_norm(gate, w, up)[1], [gate, w, up])):
        assert y.shape == gate.shape
        for g, t in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
            assert g.shape == t.shape and not g.any()
    weight = torch.ones(6, cols, dtype=dtype, device=DEV, requires_grad=True)
    for packed in (None, F.pack8(gate)):
        y = F.linear8(gate, weight, packed)
        assert y.shape == (*rows, 6) and not y.any()
        gx, gw = torch.autograd.grad(y, [gate, weight], torch.ones_like(y))
        assert gx.shape == gate.shape and gw.shape == weight.shape and not gw.any()
    assert F.checkpoint8(torch.nn.Identity(), gate).shape == gate.shape


def test_forward_mode_derivatives():
    """Refused by the operators that do not carry them on, right through linear8's plain product."""
    import torch.autograd.forward_ad as forward

    x, t, w = randn(1, 5, 64), randn(2, 5, 64), randn(3, 40, 64)
    with forward.dual_level():
        dual = forward.make_dual(x, t)
        for call in (lambda: F.rms_norm(dual, w[0]), lambda: F.rms_norm8(x, w[0], dual), lambda: F.gated_silu(x, dual), lambda: F.gated_silu8(dual)):
            with pytest.raises(RuntimeError, match="forward-mode derivatives are not supported"):
                call()
        assert torch.equal(forward.unpack_dual(F.linear8(dual, w)).tangent, F.linear8(t, w))
        for call in (lambda: F.linear8(dual, w.requires_grad_()), lambda: F.checkpoint8(torch.nn.Linear(64, 3).to(DEV), dual)):
            with pytest.raises(RuntimeError, match="jvp|forward AD"):
                call()


@pytest.mark.parametrize("cols", [1, 31, 64, 500, 4096, 33000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_whose_output_has_no_gradient(dtype, cols):
    """Only h is used: the gradient is h's own, bit for bit, whatever h and the weight hold, and the weight's is zero."""
    x, r, w = randn(1, 6, cols, dtype=dtype), randn(2, 6, cols, dtype=dtype), randn(3, cols, dtype=dtype)
    x[1, 0], x[2, cols // 2], r[3, cols - 1], w[cols // 2] = float("inf"), float("nan"), -float("inf"), float("inf")
    for t in (x, r, w):
        t.requires_grad_()
    gh = randn(4, 6, 2 * cols, dtype=dtype)[:, cols:]
    for f in (lambda: F.rms_norm(x, w, r)[1], lambda: F.rms_norm8(x, w, r).h):
        gx, gr, gw = torch.autograd.grad(f(), [x, r, w], gh)
        assert torch.equal(gx, gh) and torch.equal(gr, gh) and torch.equal(gw, torch.zeros_like(w))


def test_abi_norm_backward_without_gradients():
    """grad_y and grad_h both null: zeros."""
    from morphocore_amd import _native

    h, w, rstd = randn(1, 5, 77), randn(2, 77), torch.full((5,), float("nan"), device=DEV)
    gx, gw = torch.full((5, 77), 7.0, device=DEV), torch.full((77,), 7.0, device=DEV)
    lib = _native.lib()
    need = lib.mca_rms_norm_backward_workspace_size(5, 77)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    rc = lib.mca_rms_norm_backward(0, 0, None, 0, None, 0, h.data_ptr(), 77, w.data_ptr(), rstd.data_ptr(), gx.data_ptr(), gw.data_ptr(), 5, 77,
                                   ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and not gx.any() and not gw.any()


@pytest.mark.parametrize("cols", [3, 64, 500, 4096, 33000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_of_weights_and_rows_that_are_not_finite(dtype, cols):
    """y is h * rstd * weight, infinite where the weight is and NaN only where that is NaN: an infinite weight on a zero, a NaN weight,
    a row with an infinity (rstd 0) or a NaN."""
    x, w = randn(1, 7, cols, dtype=dtype), randn(2, cols, dtype=torch.float32)
    w[0], w[cols // 2], w[cols - 1] = float("inf"), -float("inf"), float("nan")
    x[1, 0], x[2, 1], x[3, 1], x[4] = 0, float("inf"), float("nan"), 0
    for wt in (w, w.to(dtype)):
        v = x.double()
        want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6) * wt.double()
        for y in (F.rms_norm(x, wt), F.rms_norm8(x, wt).y, F.rms_norm(x, wt, torch.zeros_like(x))[0]):
            same = torch.isnan(want) == torch.isnan(y)
            assert same.all() and torch.equal(torch.isinf(want), torch.isinf(y))
            infinite = torch.isinf(want)
            assert torch.equal(y[infinite].double(), want[infinite])


def test_checkpoint_of_a_module_that_writes_to_its_input():
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.LeakyReLU(0.1, inplace=True), torch.nn.Linear(64, 48)).to(DEV)
    x, gy = F.unpack8(F.pack8(randn(1, 9, 64))), randn(2, 9, 48)  # values that a checkpoint holds exactly
    results = []
    for call in (net, lambda t: F.checkpoint8(net, t)):
        a = x.clone().requires_grad_()
        b = a * 1.0
        out = call(b)
        got = [b, out, *torch.autograd.grad([out, b], [a, *net.parameters()], [gy, x])]
        out = call(x.clone())
        results.append([*got, *torch.autograd.grad(out, net.parameters(), gy)])
    for plain, kept in zip(*results):
        assert torch.equal(plain, kept)


@pytest.mark.parametrize("rows,cols", [(1, 40), (2000, 777), (50, 4096), (7, 33000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_norm_gradients_against_the_unrounded_sum(dtype, rows, cols):
    """The backward reads h as stored: its gradients are those of the sum x + residual that the forward normalised but for h's
    rounding, at most u of each h.

    Elementwise, with u the unit roundoff: u of the sum of the terms' magnitudes in the weight's gradient and twice u of n's share
    in the input's, besides the bounds of the gradients at the stored h (64 units of 2^-24 of the terms, sums over rows
    2 sqrt(rows) + 16, the output's u). Over all of the weight's gradient, two independent roundings of at most u / sqrt(3)
    by norm each (h's and the output's): sqrt(2 / 3) u.
    """
    u, f = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype], 2.0**-24
    x, r, w = randn(1, rows, cols, dtype=dtype).requires_grad_(), randn(2, rows, cols, dtype=dtype), (1 + 0.2 * randn(3, cols)).to(dtype).requires_grad_()
    gy = randn(4, rows, cols, dtype=dtype, scale=0.1)
    y, h = F.rms_norm(x, w, r, 1e-5)
    gx, gw = torch.autograd.grad(y, [x, w], gy)
    s, a = x.detach().double() + r.double(), gy.double() * w.detach().double()
    rstd = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-5)
    n = s * rstd
    want = rstd * (a - n * (a * n).mean(-1, keepdim=True))
    share = rstd * n.abs() * (a * n).abs().mean(-1, keepdim=True)
    size = 64 * f * (rstd * a.abs() + share) + (2 * u + u * u) * share
    assert ((gx.double() - want).abs() <= size + u * (want.abs() + size) + 2.0**-25).all()
    terms = gy.double() * n
    want, size = terms.sum(0), (u + (2 * np.sqrt(rows) + 16) * f) * terms.abs().sum(0)
    assert ((gw.double() - want).abs() <= size + u * (want.abs() + size) + 2.0**-25).all()
    if rows >= 50:
        assert (gw.double() - want).norm() <= np.sqrt(2 / 3) * u * want.norm()


@pytest.mark.parametrize("cols", [16384, 16385, 32801, 100003, 500009])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_of_the_widest_rows(dtype, cols):
    """A lane's sum has 8 ceil(units / 1024) terms, which grows with the width: the sum of squares is off by that many units
    of 2^-24 and 10 of the tree, half of which the root leaves; 8 more for the root, the division and the products. float16's
    subnormal results add half their spacing."""
    f, u = 2.0**-24, {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    half_spacing = 2.0**-25 if dtype == torch.float16 else 0.0
    x, r, w = randn(1, 3, cols, dtype=dtype), randn(2, 3, cols, dtype=dtype), (1 + 0.2 * randn(3, cols)).to(dtype)
    s = x.double() + r.double()
    want = s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    terms = 8 * -(-(-(-cols // 8)) // 1024)
    y, h = F.rms_norm(x, w, r)
    # The float32 sum x + residual rounds once more.
    far = (y.double() - want).abs() - (((terms + 10) / 2 + 8) * f + u) * want.abs() - f * (x.double().abs() + r.double().abs())
    assert (far[want.abs() >= 2.0**-14] <= 0).all() and (far <= half_spacing).all()
    assert torch.equal(h, (x.float() + r.float()).to(dtype))


@pytest.mark.parametrize("rows,cols", [(300, 64), (200, 500), (50, 4096), (20, 16384), (9, 33000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_norm_rounds_its_output_once(dtype, rows, cols):
    """y is (x + residual, in float32) * rstd * weight rounded to float32 and then to its type.

    What comes before the first rounding: the sum of squares in float64; rstd in two float32 terms, a Newton step from one within 2^-22
    (its square, 2^-44); their products with v and the weight with the errors carried along, which round once more at 2^-24
    of 2^-22 each: below 2^-42 in all. float16's subnormal results add half their spacing.
    """
    f, first = 2.0**-24, 2.0**-24 + 2.0**-42
    u = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    x, r = randn(1, rows, cols, dtype=dtype) * torch.exp(randn(2, rows, 1)).to(dtype), randn(3, rows, cols, dtype=dtype)
    w = (1 + 0.2 * randn(4, cols)).to(dtype)
    eps = float(np.float32(1e-6))
    for residual in (None, r):
        v = (x.float() if residual is None else x.float() + r.float()).double()
        want = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()
        y = F.rms_norm(x, w, residual, eps)
        y = (y if residual is None else y[0]).double()
        spacing = torch.where(want.abs() < 2.0**-14, 2.0**-25, 0.0) if dtype == torch.float16 else 0.0
        assert ((y - want).abs() <= (first + u * (1 + first)) * want.abs() + spacing).all()
        # Another value than the rounded float64 one only where the first rounding ends at a midpoint of the type's values: one in 2^13
        # of float16 and 2^16 of bfloat16 at most, by half a step of float32 each way; four times that many are allowed.
        if dtype != torch.float32:
            assert (y != want.to(dtype).double()).double().mean() <= 4 * f / u
