"""Every shape of linear attention's walk over the chunks (tests/walk_cases.py) against float64 (tests/tokens_torch.py).

Tolerance, of the sum M of the terms' magnitudes with every decay's reach counted in, f = 2^-24: products of dim terms and sums over the tokens
2 sqrt(dim) + 2 sqrt(tokens) + 64 units f; operands, scores and states are held in three terms of 8 bits (16-bit operands exactly), and what
products of them leave out is below 4 f, within the 64. The result's rounding adds eps / 2 of the value, or half a subnormal's spacing."""
import math

import pytest
import torch

import morphocore_amd.functional as F
from tests import tokens_torch as T
from tests.walk_cases import CASES

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
RUNS = [(c, t) for c in CASES for t in c["types"]]


def name_of(run):
    c, t = run
    return (f"{str(TYPES[t])[6:]}-{c['dim']}x{c['value_dim']}-{c['sequences']}x{sum(c['lengths'])}{'packed' if c['packed'] else ''}-"
            f"{c['heads'] * c['copies']}of{c['kv_heads'] * c['copies']}-{'train' if c['train'] else 'forward'}")


def data(c, dtype):
    """The sequences once: q, k, v, go [rows, heads, .], first and last states, decays."""
    g = torch.Generator().manual_seed(c["dim"] * 1000 + c["value_dim"])
    rand = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    n, heads, kv, dim, dv = sum(c["lengths"]), c["heads"], c["kv_heads"], c["dim"], c["value_dim"]
    rows = [rand(n, h, d).to(DEV, dtype) for h, d in ((heads, dim), (kv, dim), (kv, dv), (heads, dv))]
    states = [rand(len(c["lengths"]), heads, dim, dv).to(DEV) for _ in range(2)]
    decays = torch.log1p(-torch.exp2(-torch.tensor([3.0, 9.0, 6.0, 11.0]))).to(DEV)[:heads].clone()
    decays[-1] = 0.0
    return rows, states, decays


def run(c, rows, states, decays, scale):
    """The call with the data's copies, and every result folded back to [sequences, rows or states, copies, heads, ..]."""
    s, copies = c["sequences"], c["copies"]
    n, count = sum(c["lengths"]), len(c["lengths"])
    spread = [t.repeat(s, copies, 1) if c["packed"] else t.repeat(1, copies, 1).expand(s, *t.repeat(1, copies, 1).shape).contiguous() for t in rows]
    q, k, v, go = spread
    first, last = (t.repeat(s, copies, 1, 1) for t in states)
    offsets = None
    if c["packed"]:
        offsets = torch.tensor([0, *(c["lengths"] * s)], device=DEV).cumsum(0)
    g = decays.repeat(copies)
    if c["train"]:
        leaves = [t.requires_grad_() for t in (q, k, v, first)]
        out, state = F.linear_attention(q, k, v, g, first, offsets, scale, True)
        got = dict(zip(("out", "state", "gq", "gk", "gv", "gs"), (out.detach(), state.detach(), *torch.autograd.grad([out, state], leaves, [go, last]))))
    else:
        with torch.no_grad():
            got = dict(zip(("out", "state"), F.linear_attention(q, k, v, g, first, offsets, scale, True)))
    for name, t in got.items():
        heads = c["kv_heads"] if name in ("gk", "gv") else c["heads"]
        got[name] = t.reshape(s, count if name in ("state", "gs") else n, copies, heads, *t.shape[-2 if name in ("state", "gs") else -1:])
    return got


def near(got, want, size, what):
    far = (got.double() - want).abs()
    bad = ~(far <= size + torch.finfo(got.dtype).eps / 2 * want.abs() + TINY[got.dtype])
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values, first {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}"


@pytest.mark.parametrize("case", RUNS, ids=map(name_of, RUNS))
def test_walk(case):
    c, kind = case
    rows, states, g = data(c, TYPES[kind])
    scale = c["dim"]**-0.5
    got = run(c, rows, states, g, scale)
    for name, t in got.items():
        one = t[0, :, 0]
        assert torch.equal(t, one[None, :, None].expand_as(t)), f"{name}: copies of the same data differ"
    at, share = 0, c["heads"] // c["kv_heads"]
    for i, n in enumerate(c["lengths"]):
        r = slice(at, at + n)
        at += n
        q, k, v, go = (t[r] for t in rows)
        want = T.attention(q, k, v, g, scale, states[0][i], *((go, states[1][i]) if c["train"] else ()))
        f = (2 * math.sqrt(max(c["dim"], c["value_dim"]) * share) + 2 * math.sqrt(n) + 64) * 2.0**-24
        for name, t in got.items():
            near(t[0, i, 0] if name in ("state", "gs") else t[0, r, 0], want[name][0], f * want[name][1], f"sequence {i} {name}")


SPOILED = [(c, t) for c, t in RUNS if c["copies"] > 1 and not c["packed"]]


@pytest.mark.parametrize("value", ["inf", "nan"])
@pytest.mark.parametrize("case", SPOILED, ids=map(name_of, SPOILED))
def test_walks_of_much_work_keep_what_is_not_finite_apart(case, value):
    """Of a value: its column of out from its row on, and of the state; the other results stay the same bits. Of a key likewise, in every column."""
    c, kind = case
    rows, states, g = data(c, TYPES[kind])
    at, col = sum(c["lengths"]) // 2 + 3, 5
    want = run(c, rows, states, g, 0.1)
    for which in (1, 2):
        bad = [t.detach().clone() for t in rows]
        bad[which][at, 0, col] = float(value)
        got = run(c, bad, [t.detach().clone() for t in states], g, 0.1)
        hit = {name: torch.zeros_like(t, dtype=torch.bool) for name, t in want.items()}
        own = slice(0, c["heads"] // c["kv_heads"])  # the heads that share it
        if which == 2:
            hit["out"][:, at:, :, own, col], hit["state"][:, :, :, own, :, col] = True, True
        else:
            hit["out"][:, at:, :, own], hit["state"][:, :, :, own, col] = True, True
        if c["train"]:
            if which == 2:
                hit["gq"][:, at:, :, own], hit["gk"][:, at, :, 0] = True, True
            else:
                hit["gq"][:, at:, :, own, col], hit["gv"][:, at, :, 0] = True, True
        for name, t in got.items():
            assert not torch.isfinite(t[hit[name]]).any(), f"{which} {name}: finite where it depends"
            assert torch.equal(t[~hit[name]], want[name][~hit[name]]), f"{which} {name}: changed elsewhere"
