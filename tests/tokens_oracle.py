"""The token-mixing operators in numpy float64, from their definitions: rotations as complex products, the norm of a head's row,
linear attention by every pair of tokens. Results come with the sum of their terms' magnitudes, which scales their error."""
import numpy as np


def angles(positions, frequencies):
    """[tokens, pairs] of positions [tokens, axes]."""
    return positions.astype(np.float64) @ frequencies


def pairs_of(x, n, interleaved):
    """The pairs' first and second values, as views."""
    return (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n])


def rotate(x, angle, interleaved):
    """x [.., tokens, heads, dim] by angle [tokens, pairs]."""
    y = x.copy()
    a, b = pairs_of(x, angle.shape[-1], interleaved)
    z = (a + 1j * b) * np.exp(1j * angle)[..., None, :]
    ya, yb = pairs_of(y, angle.shape[-1], interleaved)
    ya[...], yb[...] = z.real, z.imag
    return y


def pair_size(x, n, interleaved):
    """|a| + |b| at both values of a pair, |x| behind the pairs."""
    y = np.abs(x)
    a, b = pairs_of(y, n, interleaved)
    s = a + b
    a[...], b[...] = s, s
    return y


def norm(x, w, eps):
    return x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * w


def norm_grads(x, w, eps, g):
    r = 1 / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    m, t = x * r, g * w
    return r * (t - m * np.mean(t * m, axis=-1, keepdims=True)), (g * m).reshape(-1, x.shape[-1]).sum(0)


def norm_sizes(x, w, eps, size):
    """The same of magnitudes: size of g's error."""
    r = 1 / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    m, t = np.abs(x * r), size * np.abs(w)
    return r * (t + m * np.mean(t * m, axis=-1, keepdims=True)), (size * m).reshape(-1, x.shape[-1]).sum(0)


def _weights(g, n):
    at = np.arange(n)
    gap = at[:, None] - at
    with np.errstate(over="ignore", invalid="ignore"):
        e = np.where(gap == 0, 1.0, np.exp(np.where(gap > 0, g * np.maximum(gap, 1), 0.0)))
        reach = np.where(gap > 0, np.nan_to_num(np.abs(g) * gap * e, posinf=0.0), 0.0)
    return np.where(gap >= 0, e, 0.0), reach


def power(g, n):
    """exp(g n), 1 for n = 0 whatever g."""
    n = np.asarray(n, np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(n == 0, 1.0, np.exp(np.where(n == 0, 0.0, g * n)))


def attention(q, k, v, g, scale, first=None, go=None, last=None):
    """One sequence: q [n, heads, dim], k, v [n, kv heads, .], g [heads]; first, last [heads, dim, value dim]. A dict of results, each
    (value, sum of magnitudes with the reach of every decay in it)."""
    n, heads, dim = q.shape
    kvh, dv = v.shape[1:]
    share = heads // kvh
    first = np.zeros((heads, dim, dv)) if first is None else first
    last = np.zeros((heads, dim, dv)) if last is None else last
    at = np.arange(n)
    names = ["out", "state"] + (["gq", "gk", "gv", "gs"] if go is not None else [])
    shape = {"out": (n, heads, dv), "state": first.shape, "gq": q.shape, "gk": k.shape, "gv": v.shape, "gs": first.shape}
    got = {x: [np.zeros(shape[x]), np.zeros(shape[x])] for x in names}

    def put(name, where, value, size):
        got[name][0][where] += value
        got[name][1][where] += size

    for h in range(heads):
        Q, K, V, S, L = q[:, h], k[:, h // share], v[:, h // share], first[h], last[h]
        w, reach = _weights(g[h], n)
        far, near, whole = power(g[h], at + 1)[:, None], power(g[h], n - 1 - at)[:, None], power(g[h], n)
        # A decay's own error grows with what is taken of it.
        rel = lambda e: 1 + np.abs(np.nan_to_num(np.log(np.maximum(e, 1e-300))))  # noqa: E731
        wide = w + reach
        a = np.abs
        put("out", np.s_[:, h], scale * ((Q @ K.T * w) @ V + far * (Q @ S)), scale * ((a(Q) @ a(K).T * wide) @ a(V) + far * rel(far) * (a(Q) @ a(S))))
        put("state", np.s_[h], (near * K).T @ V + whole * S, (near * rel(near) * a(K)).T @ a(V) + whole * rel(whole) * a(S))
        if go is None:
            continue
        G = go[:, h]
        gw, gwide = (G @ V.T) * w, (a(G) @ a(V).T) * wide
        put("gq", np.s_[:, h], scale * (gw @ K + far * (G @ S.T)), scale * (gwide @ a(K) + far * rel(far) * (a(G) @ a(S).T)))
        put("gk", np.s_[:, h // share], scale * gw.T @ Q + near * (V @ L.T), scale * gwide.T @ a(Q) + near * rel(near) * (a(V) @ a(L).T))
        put("gv", np.s_[:, h // share], scale * (Q @ K.T * w).T @ G + near * (K @ L), scale * (a(Q) @ a(K).T * wide).T @ a(G) + near * rel(near) * (a(K) @ a(L)))
        put("gs", np.s_[h], whole * L + scale * (far * Q).T @ G, whole * rel(whole) * a(L) + scale * (far * rel(far) * a(Q)).T @ a(G))
    return {x: tuple(y) for x, y in got.items()}


def recurrence(q, k, v, g, scale, first):
    """The definition, token after token: (out, state)."""
    n, heads, _ = q.shape
    share = heads // k.shape[1]
    s, out = first.copy(), np.zeros((n, heads, v.shape[2]))
    for t in range(n):
        for h in range(heads):
            s[h] = np.exp(g[h]) * s[h] + np.outer(k[t, h // share], v[t, h // share])
            out[t, h] = scale * q[t, h] @ s[h]
    return out, s
