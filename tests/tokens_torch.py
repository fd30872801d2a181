"""One sequence of linear attention by every pair of tokens in float64 on its tensors' device, for sequences that are too long for numpy;
tests/test_tokens_torch.py holds it to tests/tokens_oracle.py."""
import torch


def decay(g, distance):
    """exp(g distance), 1 for a distance of 0 and 0 below it; and the same with its own error's growth, 1 + |log| of it."""
    g = float(g)
    e = torch.where(distance > 0, torch.exp(g * distance.clamp(min=1)), (distance == 0).double())
    reach = torch.where(distance > 0, (abs(g) * distance.clamp(min=1) * e).nan_to_num(nan=0.0, posinf=0.0), 0.0)
    return e, e + reach


def attention(q, k, v, g, scale, first, go=None, last=None):
    """q [n, heads, dim], k, v [n, kv heads, .], first, last [heads, dim, value dim]: name -> (value, sum of magnitudes)."""
    q, k, v, g, first = (t.detach().double() for t in (q, k, v, g, first))
    n, heads, _ = q.shape
    share = heads // k.shape[1]
    train = go is not None
    zeros = lambda t, *shape: [t.new_zeros(shape) for _ in range(2)]  # noqa: E731
    got = {"out": zeros(q, n, heads, v.shape[2]), "state": zeros(q, *first.shape)}
    if train:
        go, last = go.detach().double(), last.detach().double()
        got.update(gq=zeros(q, *q.shape), gk=zeros(q, *k.shape), gv=zeros(q, *v.shape), gs=zeros(q, *first.shape))
    at = torch.arange(n, dtype=torch.float64, device=q.device)
    for h in range(heads):
        w = decay(g[h], at[:, None] - at)
        far, near = decay(g[h], at[:, None] + 1), decay(g[h], n - 1 - at[:, None])
        whole = decay(g[h], torch.full((1, 1), float(n), dtype=torch.float64, device=q.device))
        c = h // share
        given = [t.contiguous() for t in ((q[:, h], k[:, c], v[:, c], first[h]) + ((go[:, h], last[h]) if train else ()))]
        for i, (Q, K, V, S, *rest) in enumerate((given, [t.abs() for t in given])):  # the values, then their magnitudes
            score = (Q @ K.t()) * w[i]
            got["out"][i][:, h] += scale * (score @ V + far[i] * (Q @ S))
            got["state"][i][h] += (near[i] * K).t() @ V + whole[i] * S
            if train:
                G, L = rest
                gw = (G @ V.t()) * w[i]
                got["gq"][i][:, h] += scale * (gw @ K + far[i] * (G @ S.t()))
                got["gk"][i][:, c] += scale * (gw.t() @ Q) + near[i] * (V @ L.t())
                got["gv"][i][:, c] += scale * (score.t() @ G) + near[i] * (K @ L)
                got["gs"][i][h] += whole[i] * L + scale * (far[i] * Q).t() @ G
                del gw
            del score
    return {name: tuple(pair) for name, pair in got.items()}
