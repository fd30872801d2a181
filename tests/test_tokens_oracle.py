"""The float64 oracle of the token-mixing operators against their definitions, token after token, and central differences."""
import numpy as np
import pytest

from tests import tokens_oracle as O


def draw(seed, n=7, heads=4, kvh=2, dim=5, dv=3):
    r = np.random.default_rng(seed)
    q, k, v = r.normal(size=(n, heads, dim)), r.normal(size=(n, kvh, dim)), r.normal(size=(n, kvh, dv))
    return q, k, v, np.log(r.uniform(0.3, 0.99, heads)), 0.4, r.normal(size=(heads, dim, dv)), r.normal(size=(n, heads, dv)), r.normal(size=(heads, dim, dv))


@pytest.mark.parametrize("n", [0, 1, 2, 9])
def test_attention_is_the_recurrence(n):
    q, k, v, g, scale, first, _, _ = draw(1, n)
    got = O.attention(q, k, v, g, scale, first)
    out, state = O.recurrence(q, k, v, g, scale, first)
    assert np.allclose(got["out"][0], out, rtol=1e-12, atol=1e-12) and np.allclose(got["state"][0], state, rtol=1e-12, atol=1e-12)
    assert (got["out"][1] >= np.abs(out) * (1 - 1e-12)).all() and (got["state"][1] >= np.abs(state) * (1 - 1e-12)).all()


def test_attention_without_memory_and_without_decay():
    q, k, v, _, scale, first, _, _ = draw(2)
    got = O.attention(q, k, v, np.array([-np.inf, 0.0, -np.inf, 0.0]), scale, first)
    for h, want in ((0, np.zeros((5, 3))), (1, first[1])):
        s = want
        for t in range(len(q)):
            s = np.outer(k[t, 0], v[t, 0]) + (s if h == 1 else 0)
            assert np.allclose(got["out"][0][t, h], scale * q[t, h] @ s)
        assert np.allclose(got["state"][0][h], s)


def test_attention_gradients_by_differences():
    q, k, v, g, scale, first, go, last = draw(3)
    grads = O.attention(q, k, v, g, scale, first, go, last)

    def loss():
        r = O.attention(q, k, v, g, scale, first)
        return (r["out"][0] * go).sum() + (r["state"][0] * last).sum()

    for name, x in (("gq", q), ("gk", k), ("gv", v), ("gs", first)):
        for i in np.ndindex(x.shape):
            kept, step = x[i], 1e-5
            x[i] = kept + step
            up = loss()
            x[i] = kept - step
            down = loss()
            x[i] = kept
            assert abs((up - down) / (2 * step) - grads[name][0][i]) < 1e-7


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_and_norm(interleaved):
    r = np.random.default_rng(4)
    x, w, angle, gy = r.normal(size=(3, 2, 9)), r.normal(size=9), r.normal(size=(3, 4)), r.normal(size=(3, 2, 9))
    y = O.rotate(x, angle, interleaved)
    for t in range(3):
        for j in range(4):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, 4 + j)
            c, s = np.cos(angle[t, j]), np.sin(angle[t, j])
            assert np.allclose(y[t, :, a], x[t, :, a] * c - x[t, :, b] * s) and np.allclose(y[t, :, b], x[t, :, b] * c + x[t, :, a] * s)
    assert np.array_equal(y[..., 8], x[..., 8]) and np.allclose(O.rotate(y, -angle, interleaved), x)
    gx, gw = O.norm_grads(x, w, 1e-3, O.rotate(gy, -angle, interleaved))
    loss = lambda: (O.rotate(O.norm(x, w, 1e-3), angle, interleaved) * gy).sum()  # noqa: E731
    for value, grad in ((x, gx), (w, gw)):
        for i in np.ndindex(value.shape):
            kept, step = value[i], 1e-5
            value[i] = kept + step
            up = loss()
            value[i] = kept - step
            down = loss()
            value[i] = kept
            assert abs((up - down) / (2 * step) - grad[i]) < 1e-7
