"""nn.TokenMixer on the GPU: against its formulas in float64, and its forms against each other."""
import importlib.util
import os

import pytest
import torch

import morphocore_amd.functional as F
import morphocore_amd.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda"


def randn(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def mixer(channels, heads, **kw):
    torch.manual_seed(0)
    m = nn.TokenMixer(channels, heads, **kw).to(DEV)
    with torch.no_grad():
        for p in (m.norm.weight, m.query_weight, m.key_weight):
            p.add_(0.2 * torch.randn_like(p))
    return m


def formulas(m, x, residual, positions, state):
    """The module's outputs of [batch, tokens, channels] on the CPU; x and the parameters (a name's tensor) in float64."""
    p = {name: t.detach().double().cpu().requires_grad_() for name, t in m.named_parameters()}
    h = x + residual

    def normed(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.norm.eps) * w

    joint = (normed(h, p["norm.weight"]) @ p["project"].t()).unflatten(-1, (m.heads + 2 * m.kv_heads, m.dim))
    q, k, v = joint.split((m.heads, m.kv_heads, m.kv_heads), -2)
    angle = (positions.cpu().double() @ m.frequencies.cpu())[:, None]
    n = angle.shape[-1]

    def turned(t):
        a, b, rest = t.split((n, n, t.shape[-1] - 2 * n), -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest], -1)

    share = m.heads // m.kv_heads
    q, k = turned(normed(q, p["query_weight"])).movedim(-2, 1), turned(normed(k, p["key_weight"])).repeat_interleave(share, -2).movedim(-2, 1)
    v, g = v.repeat_interleave(share, -2).movedim(-2, 1), m.log_decay.double().cpu()[:, None, None]
    at = torch.arange(x.shape[1], dtype=torch.float64)
    gap = at[:, None] - at
    weight = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0)
    out = ((q @ k.transpose(-1, -2)) * weight @ v + torch.exp(g * (at[:, None] + 1)) * (q @ state)) * m.dim**-0.5
    last = torch.exp(g * len(at)) * state + k.transpose(-1, -2) @ (torch.exp(g * (at[-1] - at[:, None])) * v)
    return p, out.movedim(1, -2).flatten(-2) @ p["contract"].t(), h, last


@pytest.mark.parametrize("kv_heads,dim", [(4, 16), (2, 21)])
def test_against_float64(kv_heads, dim):
    """Outputs: five operators in turn, each below 2^-17 of its terms; gradients within 1/16 by norm, the most that a kept value may be off."""
    m = mixer(40, 4, axes=2, kv_heads=kv_heads, dim=dim)
    x, r, s = randn(1, 2, 9, 10, 40).requires_grad_(), randn(2, 2, 9, 10, 40).requires_grad_(), randn(3, 2, 4, dim, dim).requires_grad_()
    gradients = randn(4, 2, 9, 10, 40), randn(5, 2, 9, 10, 40), randn(6, 2, 4, dim, dim)
    got = m(x, r, state=s, final_state=True)
    grads = torch.autograd.grad(got, [x, r, s, *m.parameters()], gradients)
    x64, r64, s64 = (t.detach().double().cpu().requires_grad_() for t in (x, r, s))
    p, *want = formulas(m, x64.flatten(1, 2), r64.flatten(1, 2), F.grid_positions([9, 10]), s64)
    for a, b in zip(got, want):
        assert (a.double().cpu().reshape(b.shape) - b).norm() <= 2.0**-15 * b.norm()
    want = torch.autograd.grad(want, [x64, r64, s64, *p.values()], [g.double().cpu().reshape(w.shape) for g, w in zip(gradients, want)])
    assert [n for n, _ in m.named_parameters()] == list(p)
    for a, b in zip(grads, want):
        assert (a.double().cpu() - b).norm() <= b.norm() / 16


def test_images_as_the_morphological_layers_hold_them():
    m, first = mixer(32, 2, axes=2), mixer(32, 2, axes=2, channels_first=True)
    x, r = randn(1, 2, 32, 5, 7), randn(2, 2, 32, 5, 7)
    out, h = first(x, r)
    want, _ = m(x.permute(0, 2, 3, 1), r.permute(0, 2, 3, 1))
    assert torch.equal(h, x + r) and torch.equal(out, want.permute(0, 3, 1, 2)) and out.is_contiguous()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_packed_prompts_then_steps(dtype):
    """Packed sequences as each alone, then tokens one by one as the sequence that holds them. Each form rounds its intermediate
    results to the type (unit u: 2^-24, 2^-11, 2^-8) by itself, seven times, every one below 2 u of the next by norm: 16 u, and for the
    sums of the products in float32 as much again."""
    lengths, more = [7, 0, 70, 1], 3
    m = mixer(32, 4, kv_heads=2, dtype=dtype)
    assert m.log_decay.dtype == torch.float32 and m.frequencies.dtype == torch.float64
    whole = [randn(i, n + more, 32, dtype=dtype) for i, n in enumerate(lengths)]
    with torch.no_grad():
        want = [m(w[None])[0][0] for w in whole]
        at = torch.cat([torch.arange(n, device=DEV) for n in lengths])[:, None]
        offsets = torch.tensor([0, 7, 7, 77, 78], device=DEV)
        out, h, last = m(torch.cat([w[:n] for w, n in zip(whole, lengths)]), positions=at, offsets=offsets, final_state=True)
        cache, slots = torch.zeros(6, 4, 8, 8, device=DEV), torch.tensor([4, 1, 5, 0], device=DEV)
        cache[slots] = last
    steps = []
    for i in range(more):
        x = torch.stack([w[n + i] for w, n in zip(whole, lengths)])
        y, h = m.step(x, cache, torch.tensor(lengths, device=DEV)[:, None] + i, torch.zeros_like(x), slots)
        assert not y.requires_grad and torch.equal(h, x)
        steps.append(y)
    u = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    for i, w in enumerate(want):
        got = torch.cat([out[offsets[i]:offsets[i + 1]], torch.stack([s[i] for s in steps])])
        assert (got.float() - w.float()).norm() <= 32 * u * w.float().norm(), f"sequence {i}"


def test_inference_and_autocast():
    """The same bits as otherwise, and a state of either kind written in place."""
    m = mixer(32, 4, axes=2)
    x = randn(1, 2, 3, 5, 32)
    want = m(x, final_state=True)
    at, state = torch.tensor([[3, 0], [1, 2]], device=DEV), want[2].detach().clone()
    token = m.step(x[:, 0, 0], state, at)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = m(x, final_state=True)
        other = want[2].detach().clone()
        assert torch.equal(m.step(x[:, 0, 0], other, at)[0], token[0]) and torch.equal(other, state)
    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))
    r = randn(2, 2, 3, 5, 32)
    with torch.no_grad():
        got = m(x, final_state=True), m(x, r)
    assert all(torch.equal(a, b) for a, b in zip((*got[0], *got[1]), (*want, *m(x, r))))
    with torch.inference_mode():
        got = m(x, final_state=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for other in (want[2].detach().clone(), got[2]):
            assert torch.equal(m.step(x[:, 0, 0], other, at)[0], token[0]) and torch.equal(other, state)


@pytest.mark.parametrize("shape", [(0, 3, 5), (2, 0, 5), (2, 1, 1)])
def test_no_tokens(shape):
    m = mixer(32, 4, axes=2)
    x, s = randn(1, *shape, 32).requires_grad_(), randn(2, shape[0], 4, 8, 8)
    out, h, last = m(x, state=s, final_state=True)
    assert out.shape == h.shape == x.shape and last.shape == s.shape
    if x.numel() == 0:
        assert torch.equal(last, s)
    grads = torch.autograd.grad([out, last], [x, *m.parameters()], [torch.ones_like(out), torch.ones_like(last)], allow_unused=True)
    assert all(g is None or torch.isfinite(g).all() for g in grads)


def test_captured_training_step():
    """A step's forward and backward in a graph, each replay as the eager step."""
    m = mixer(32, 4, axes=2)
    x, go = randn(1, 2, 6, 7, 32).requires_grad_(), randn(2, 2, 6, 7, 32)

    def step():
        out, h = m(x)
        return [out.detach(), *torch.autograd.grad(out, [x, *m.parameters()], go)]

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
    for i in range(3):
        with torch.no_grad():
            x.copy_(randn(10 + i, 2, 6, 7, 32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b) or (a - b).norm() <= 1e-6 * b.norm(), f"replay {i}"


def test_captured_step():
    m = mixer(32, 4)
    x, cache, at = randn(1, 3, 32), randn(2, 3, 4, 8, 8), torch.tensor([[3], [0], [900]], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(x, cache, at)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = m.step(x, cache, at)
    for i in range(3):
        x.copy_(randn(10 + i, 3, 32))
        at += 1
        other = cache.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m.step(x, other, at)[0]) and torch.equal(cache, other)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_example_attends(dtype):
    """The example's network with token mixers runs, and every parameter and the image get gradients."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_mixer.py")
    spec = importlib.util.spec_from_file_location("train_mixer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, kept = example.train(steps=3, size=16, batch=2, channels=16, dtype=dtype, attend=2)
    assert all(torch.isfinite(torch.tensor(losses))) and kept > 0
    torch.manual_seed(0)
    net = example.Net(16, 2, dtype, 2).to(DEV)
    with torch.no_grad():
        net.read.add_(0.1 * torch.randn_like(net.read))
    x = randn(1, 2, 1, 16, 16, dtype=dtype).requires_grad_()
    grads = torch.autograd.grad(net(x).float().square().sum(), [x, *net.parameters()])
    assert all(torch.isfinite(g).all() and g.any() for g in grads)


def test_refusals():
    m = mixer(32, 4, axes=2)
    for bad in (lambda: m(randn(1, 2, 9, 32)), lambda: m(randn(1, 9, 32), offsets=torch.tensor([0, 9], device=DEV)),
                lambda: m(randn(1, 9, 32), positions=torch.zeros(9, 2, device=DEV)), lambda: m.step(randn(1, 2, 3, 32), None, None)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        m(randn(1, 9, 32), positions=torch.zeros(9, 1, device=DEV), offsets=torch.tensor([0, 9], device=DEV))
