"""tests/tokens_torch.py against the numpy oracle."""
import numpy as np
import pytest
import torch

from tests import tokens_oracle as O
from tests import tokens_torch as T


@pytest.mark.parametrize("n,heads,kvh", [(0, 2, 1), (1, 2, 2), (23, 4, 2)])
@pytest.mark.parametrize("train", [False, True])
def test_same_values_and_magnitudes(n, heads, kvh, train):
    r = np.random.default_rng(n)
    q, k, v = r.normal(size=(n, heads, 5)), r.normal(size=(n, kvh, 5)), r.normal(size=(n, kvh, 3))
    g = np.array([0.0, -0.3, -np.inf, -0.01])[:heads]
    first, go, last = r.normal(size=(heads, 5, 3)), r.normal(size=(n, heads, 3)), r.normal(size=(heads, 5, 3))
    want = O.attention(q, k, v, g, 0.4, first, *((go, last) if train else ()))
    t = [torch.from_numpy(x) for x in (q, k, v, g, first, go, last)]
    got = T.attention(*t[:4], 0.4, t[4], *(t[5:] if train else ()))
    assert sorted(got) == sorted(want)
    for name in want:
        for a, b in zip(got[name], want[name]):
            assert np.allclose(a.numpy(), b, rtol=1e-12, atol=1e-12), name
