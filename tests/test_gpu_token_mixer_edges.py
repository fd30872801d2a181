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
