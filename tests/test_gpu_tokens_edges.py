"""The token-mixing operators where intermediate bits, values that are not finite, layouts and launches matter."""
import pytest
import torch

import morphocore_amd.functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]

# ------------------------------------------------------------------------------------------------
# Scores and states hold float32's bits
# ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("at", [(0, 1), (20, 37), (5, 100)])
@pytest.mark.parametrize("dim,dv", [(8, 16), (16, 8), (64, 64), (128, 128), (96, 77), (256, 200)])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_and_states_keep_float32_bits(dtype, dim, dv, at):
    """Two scores (or two of a state's values) that differ in their 21st bit and cancel: 1 + 2^-9 + 2^-20 and 1 + 2^-9. Every product
    and sum is a float32, so that the result is 2^-20 exactly, as is its rounding to any of the types."""
    n, small = 110, 2.0**-20
    fine, first, second = (torch.tensor(t, device=DEV) for t in ([1, 2.0**-9, small], [1.0, 1.0, 1.0], [1.0, 1.0, 0.0]))
    g = torch.zeros(1, device=DEV)

    def call(q={}, k={}, v={}, go={}, state={}, last={}):
        """The results for operands that are zero but for the given places."""
        def filled(places, *shape, dtype=dtype):
            t = torch.zeros(*shape, device=DEV)
            for row, value in places.items():
                t[row][:len(value)] = torch.as_tensor(value, device=DEV)
            return t.to(dtype)

        rows = [filled(p, n, d)[None, :, None].detach().requires_grad_() for p, d in ((q, dim), (k, dim), (v, dv))]
        s = filled(state, 1, 1, dim, dv, dtype=torch.float32).requires_grad_()
        out, _ = got = F.linear_attention(*rows, g, s, scale=1.0, final_state=True)
        grads = torch.autograd.grad(got, rows, [filled(go, n, dv)[None, :, None], filled(last, 1, 1, dim, dv, dtype=torch.float32)])
        return [t.detach()[0, :, 0, 0].float() for t in (out, *grads)]

    a, b = at
    one, minus = [1.0], [-1.0]
    x, y, turn = [1 + 2.0**-9 + small], [1 + 2.0**-9], [1.0, -1.0]
    row = lambda d: (0, 0, d)  # noqa: E731
    assert call(q={b: fine}, k={a: first, b: second}, v={a: one, b: minus})[0][b] == small, "out, scores"
    assert call(go={b: fine}, v={a: first, b: second}, k={a: one, b: minus})[1][b] == small, "grad of q, scores"
    assert call(v={a: fine}, go={a: first, b: second}, q={a: one, b: minus})[2][a] == small, "grad of k, scores"
    assert call(k={a: fine}, q={a: first, b: second}, go={a: one, b: minus})[3][a] == small, "grad of v, scores"
    assert call(q={a: turn}, state={row(0): x, row(1): y})[0][a] == small, "out, state"
    assert call(go={a: turn}, state={row(0): x + y})[1][a] == small, "grad of q, state"
    assert call(v={a: turn}, last={row(0): x + y})[2][a] == small, "grad of k, state"
    assert call(k={a: turn}, last={row(0): x, row(1): y})[3][a] == small, "grad of v, state"


# ------------------------------------------------------------------------------------------------
# Values behind the pairs
# ------------------------------------------------------------------------------------------------


def table(axes, pairs):
    return (torch.rand(axes, pairs, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 2 - 0.3).to(DEV)


def bits(t):
    return t.detach().contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(1, 0), (5, 2), (24, 7), (40, 3), (100, 9), (200, 60), (257, 13), (512, 0), (512, 200)])
@pytest.mark.parametrize("dtype", TYPES)
def test_values_behind_the_pairs_stay_bit_for_bit(dtype, dim, pairs, interleaved):
    """Infinities, NaN and zeros of either sign behind the pairs stay, and so do their neighbours, in the result and in the gradient."""
    g = torch.Generator().manual_seed(dim)
    x, gy = (torch.randn(3, 4, dim, generator=g).to(DEV, dtype) for _ in range(2))
    p, f = torch.tensor([[0], [3], [1000]], device=DEV), table(1, pairs)
    for t in (x, gy):
        tail = t[..., 2 * pairs:]
        for i, value in enumerate((float("inf"), float("nan"), -float("inf"), -0.0, 0.0)):
            for row in range(4):
                tail[:, row, (3 * i + 5 * row) % tail.shape[-1]] = value
    clean = x.clone()
    clean[..., 2 * pairs:] = 1.0
    x.requires_grad_()
    y = F.axial_rotary(x, p, f, interleaved)
    (gx,) = torch.autograd.grad(y, x, gy)
    for got, given in ((y, x), (gx, gy)):
        assert torch.equal(bits(got[..., 2 * pairs:]), bits(given[..., 2 * pairs:]))
    assert torch.equal(y[..., :2 * pairs], F.axial_rotary(clean, p, f, interleaved)[..., :2 * pairs])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_weight_behind_the_pairs_reaches_its_own_values(value, interleaved):
    x, w, p, f = torch.randn(5, 3, 100, generator=torch.Generator().manual_seed(1)).to(DEV), torch.ones(100, device=DEV), torch.arange(5, device=DEV)[:, None], table(1, 9)
    clean = F.rms_norm_rotary(x, x, w, w, p, f, interleaved=interleaved)
    bad = w.clone()
    bad[26] = value
    for got, want in zip(F.rms_norm_rotary(x, x, bad, bad, p, f, interleaved=interleaved), clean):
        assert not torch.isfinite(got[..., 26]).any()
        got[..., 26], want[..., 26] = 0, 0
        assert torch.equal(got, want)
