"""nn.TokenMixer on the GPU: positions of every shape, and the gradients that no kept 8-bit value enters."""
import pytest
import torch

import morphocore_amd.functional as F
from tests.test_gpu_token_mixer import DEV, formulas, mixer, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [False, True])
def test_positions_of_every_shape(first):
    """The same bits for a grid's positions and for its places in one dimension, of all the batch or of each image."""
    m = mixer(32, 4, axes=2, channels_first=first)
    x = randn(1, 3, 32, 5, 6) if first else randn(1, 3, 5, 6, 32)
    at = F.grid_positions([5, 6], DEV) * 3 + 7
    want = m(x, positions=at)[0]
    assert not torch.equal(want, m(x)[0])
    for p in (at.view(5, 6, 2), at.expand(3, 30, 2), at.view(5, 6, 2).expand(3, 5, 6, 2)):
        assert torch.equal(m(x, positions=p)[0], want)
    each = torch.stack([at, at + 1, 2 * at])
    own = m(x, positions=each)[0]
    assert torch.equal(own[0], want[0]) and not torch.equal(own[1:], want[1:]) and torch.equal(m(x, positions=each.view(3, 5, 6, 2))[0], own)
    line = mixer(32, 4)
    y = randn(2, 2, 9, 32)
    assert torch.equal(line(y, positions=torch.arange(9, device=DEV)[:, None])[0], line(y)[0])
    for bad in (at[:29], at.view(6, 5, 2), at.view(5, 6, 2)[None, None].expand(1, 3, 5, 6, 2)):
        with pytest.raises(RuntimeError, match="positions must be"):
            m(x, positions=bad)


@pytest.mark.parametrize("kv_heads,dim", [(4, 16), (2, 21)])
def test_gradients_that_no_8_bit_value_enters(kv_heads, dim):
    """The gradients of the state and of the heads' norm weights: operators of float32 in turn like the outputs,
    each below 2^-17 of its terms. (The projections' weights read their kept inputs in 8 bits.)"""
    m = mixer(40, 4, axes=2, kv_heads=kv_heads, dim=dim)
    x, r, s = randn(1, 2, 9, 10, 40), randn(2, 2, 9, 10, 40), randn(3, 2, 4, dim, dim).requires_grad_()
    gradients = randn(4, 2, 9, 10, 40), randn(6, 2, 4, dim, dim)
    out, _, last = m(x, r, state=s, final_state=True)
    grads = torch.autograd.grad([out, last], [s, m.query_weight, m.key_weight], gradients)
    x64, r64, s64 = (t.detach().double().cpu().requires_grad_() for t in (x, r, s))
    p, out64, _, last64 = formulas(m, x64.flatten(1, 2), r64.flatten(1, 2), F.grid_positions([9, 10]), s64)
    want = torch.autograd.grad([out64, last64], [s64, p["query_weight"], p["key_weight"]], [g.double().cpu().reshape(w.shape) for g, w in zip(gradients, (out64, last64))])
    for a, b in zip(grads, want):
        assert (a.double().cpu() - b).norm() <= 2.0**-15 * b.norm()
