"""Cases of the token-mixing operators: rotary positions with several axes, the norm of each head's queries and
keys with the rotation in the same pass, and linear attention with a decay for each head, over whole sequences
and a token at a time.

Every case is one call as a program makes it: a training step's forward and backward (outputs and gradients), or
an inference call. With ``own`` false, ``run`` computes the operators in elementary torch operations in float32
(angles in float64); with ``own`` true, through ``morphocore_amd.functional``.

Linear attention, for each head with d = exp(log_decay): S_t = d S_(t-1) + k_t v_t^T, o_t = scale q_t S_t, scale =
1 / sqrt(key dimension). States are [.., key dimension, value dimension] float32.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
CHUNK = 128


def listed():
    return [
        # Patches of a batch of images in training: two axes, the pairs' halves apart.
        dict(name="rotary_image_train", op="rotary_train", dtype="bf16", batch=16, frames=1, height=64, width=64, heads=16, dim=64, pairs=32, interleaved=False),
        # A short video clip of odd sizes: three axes, neighbouring pairs, the row's last values left as they are.
        dict(name="rotary_video_odd", op="rotary_train", dtype="f16", batch=3, frames=5, height=27, width=31, heads=5, dim=90, pairs=39, interleaved=True),
        # One token of a served model at a far position, where only the call's latency counts.
        dict(name="norm_rotary_one_token", op="norm_rotary_infer", dtype="bf16", tokens=1, heads=32, kv_heads=8, dim=128, pairs=64, interleaved=False),
        # A training step's queries and keys, shared by groups of four heads.
        dict(name="norm_rotary_train", op="norm_rotary_train", dtype="bf16", tokens=16384, heads=32, kv_heads=8, dim=128, pairs=64, interleaved=False),
        # A ragged number of tokens, a head dimension that is no power of two, in float32.
        dict(name="norm_rotary_odd_train", op="norm_rotary_train", dtype="f32", tokens=1537, heads=6, kv_heads=3, dim=72, pairs=33, interleaved=True),
        # One long prompt.
        dict(name="attention_prompt", op="attention", dtype="bf16", batch=1, tokens=32768, heads=32, kv_heads=32, dim=128, value_dim=128, ragged=False),
        # Prompts of a server's batch, packed one after another, with heads that share keys and values and the states returned.
        dict(name="attention_ragged", op="attention", dtype="bf16", batch=41, tokens=12001, heads=16, kv_heads=4, dim=128, value_dim=128, ragged=True),
        # A training batch.
        dict(name="attention_train", op="attention_train", dtype="bf16", batch=4, tokens=4096, heads=16, kv_heads=16, dim=128, value_dim=128, ragged=False),
        # The pixels of small images with 4 heads of 16 channels in float32.
        dict(name="attention_image_train", op="attention_train", dtype="f32", batch=8, tokens=4096, heads=4, kv_heads=4, dim=16, value_dim=16, ragged=False),
        # Packed sequences of odd lengths and dimensions in float16.
        dict(name="attention_odd_train", op="attention_train", dtype="f16", batch=7, tokens=4999, heads=6, kv_heads=3, dim=96, value_dim=77, ragged=True),
        # One token of one sequence.
        dict(name="step_one", op="step", dtype="bf16", batch=1, slots=1, heads=32, kv_heads=32, dim=128, value_dim=128),
        # One token for each of a large batch, its states at their places in a cache.
        dict(name="step_batch", op="step", dtype="bf16", batch=256, slots=300, heads=32, kv_heads=32, dim=128, value_dim=128),
    ]


def _log(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return n + (rng.random() < 0.5 and n % 2 == 0 and low < n < high)


def draw(rng):
    op = rng.choice(["rotary_train", "norm_rotary_infer", "norm_rotary_train", "attention", "attention_train", "step"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    dim = rng.choice([16, 32, 64, 64, 128, 128, 256, _log(rng, 8, 256)])
    kv_heads = _log(rng, 1, 16)
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    while True:
        batch, tokens = _log(rng, 1, 64), _log(rng, 1, 32768)
        if op == "rotary_train":
            case.update(batch=batch, frames=rng.choice([1, 1, _log(rng, 2, 32)]), height=_log(rng, 2, 128), width=_log(rng, 2, 128), heads=heads, dim=dim)
            case.update(pairs=rng.choice([dim // 2, rng.randint(max(1, dim // 4), dim // 2)]), interleaved=rng.random() < 0.5)
            cost = batch * case["frames"] * case["height"] * case["width"] * heads * dim
        elif op.startswith("norm"):
            tokens = _log(rng, 1, 256) if op.endswith("infer") else tokens
            case.update(tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, pairs=rng.choice([dim // 2, rng.randint(max(1, dim // 4), dim // 2)]))
            case.update(interleaved=rng.random() < 0.5)
            cost = tokens * (heads + kv_heads) * dim
        elif op == "step":
            case.update(batch=batch, slots=batch + _log(rng, 1, 64), heads=heads, kv_heads=kv_heads, dim=dim, value_dim=rng.choice([dim, _log(rng, 8, 256)]))
            cost = batch * heads * dim * case["value_dim"] / 8
        else:
            ragged = rng.random() < 0.5
            case.update(batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, value_dim=rng.choice([dim, dim, _log(rng, 8, 256)]), ragged=ragged)
            rows = tokens if ragged else batch * tokens
            cost = max(rows * heads * max(dim, case["value_dim"]), rows * tokens * heads / 8, batch * heads * dim * case["value_dim"] / 8)
        if cost <= 2**25:
            return case


def _positions(case, g):
    """Positions [tokens, axes]: of a grid's places, or of consecutive tokens from a far one on."""
    if "frames" not in case:
        return torch.randint(100000, (1, 1), generator=g, device="cuda", dtype=torch.int32) + torch.arange(case["tokens"], device="cuda", dtype=torch.int32)[:, None]
    sizes = [case["frames"]] * (case["frames"] > 1) + [case["height"], case["width"]]
    return torch.cartesian_prod(*(torch.arange(n, device="cuda", dtype=torch.int32) for n in sizes))


def _frequencies(axes, pairs, base):
    """Radians a position, [axes, pairs] float64: each axis has its own share of the pairs, from fast to slow."""
    table = torch.zeros(axes, pairs, dtype=torch.float64, device="cuda")
    shares = [pairs // axes + (a < pairs % axes) for a in range(axes)]
    first = 0
    for axis, n in enumerate(shares):
        table[axis, first:first + n] = base ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1))
        first += n
    return table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    train = op.endswith("_train")
    state = {"op": op, "dtype": dtype}

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def input(t):
        return t.detach().requires_grad_(train)

    if op == "rotary_train":
        state["positions"] = _positions(case, g)
        tokens, axes = state["positions"].shape
        state["frequencies"] = _frequencies(axes, case["pairs"], 100.0 if axes == 2 else 10000.0)
        state["x"] = input(normal(case["batch"], tokens, case["heads"], case["dim"]))
        state["gy"] = normal(case["batch"], tokens, case["heads"], case["dim"], scale=0.05)
        state["interleaved"] = case["interleaved"]
        return state
    if op.startswith("norm"):
        tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        state["positions"] = _positions(case, g)
        state["frequencies"] = _frequencies(1, case["pairs"], 500000.0)
        # Slices of one projection, whose values follow for the attention; tokens of several sizes.
        joint = (torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g, device="cuda") * torch.exp(torch.randn(tokens, 1, generator=g, device="cuda"))).to(dtype)
        state["q"] = input(joint[:, :heads * dim].unflatten(-1, (heads, dim)))
        state["k"] = input(joint[:, heads * dim:(heads + kv_heads) * dim].unflatten(-1, (kv_heads, dim)))
        for name in ("qw", "kw"):
            state[name] = input((1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).to(dtype))
        if train:
            state["gq"], state["gk"] = normal(tokens, heads, dim, scale=0.05), normal(tokens, kv_heads, dim, scale=0.05)
        state["interleaved"] = case["interleaved"]
        return state
    heads, kv_heads, dim, value_dim, batch = case["heads"], case["kv_heads"], case["dim"], case["value_dim"], case["batch"]
    # Decays from a few tokens' reach to some thousand.
    state["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(2, 12, heads, dtype=torch.float64, device="cuda"))).float()
    if op == "step":
        rows = (batch,)
        state["state"] = torch.randn(case["slots"], heads, dim, value_dim, generator=g, device="cuda") * 3
        state["slots"] = torch.randperm(case["slots"], generator=g, device="cuda")[:batch].to(torch.int32) if case["slots"] > 1 else None
    elif case["ragged"]:
        # Lengths of very different sizes, some of them one or none.
        share = torch.exp(1.5 * torch.randn(batch, generator=g, device="cuda", dtype=torch.float64))
        ends = torch.round(torch.cumsum(share, 0) / share.sum() * case["tokens"]).to(torch.int32)
        state["offsets"] = torch.cat([ends.new_zeros(1), ends])
        state["offsets"][-1] = case["tokens"]
        rows = (case["tokens"],)
    else:
        rows = (batch, case["tokens"])
    state["q"] = input(normal(*rows, heads, dim))
    state["k"] = input(normal(*rows, kv_heads, dim))
    state["v"] = input(normal(*rows, 2 * kv_heads * value_dim)[..., kv_heads * value_dim:].unflatten(-1, (kv_heads, value_dim)))
    if train:
        state["go"] = normal(*rows, heads, value_dim, scale=0.05)
        if case["ragged"]:  # sequences that go on from a state, and into one
            state["state"] = input(torch.randn(batch, heads, dim, value_dim, generator=g, device="cuda"))
            state["gs"] = torch.randn(batch, heads, dim, value_dim, generator=g, device="cuda") * 0.05
    return state


# The plain form.


def _angles(s):
    """Cosine and sine of every token's pairs, [tokens, 1, pairs]."""
    angle = (s["positions"].double() @ s["frequencies"]).unsqueeze(1)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotated(x, cos, sin, interleaved):
    pairs = cos.shape[-1]
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else turned.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), rest], -1)


def _plain_norm_rotary(s):
    cos, sin = _angles(s)
    got = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "w"].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        got[name] = _rotated(n * w, cos, sin, s["interleaved"]).to(s["dtype"])
        if "g" + name in s:
            g = _rotated(s["g" + name].float(), cos, -sin, s["interleaved"])
            gn = g * w
            got["g" + name] = (r * (gn - n * (gn * n).mean(-1, keepdim=True))).to(s["dtype"])
            got["g" + name + "w"] = (g * n).sum((0, 1)).to(s["dtype"])
    return got


def _decay(log_decay, distance):
    """exp(log_decay * distance), [heads, ..]; 0 where the distance is negative."""
    d = distance.to(log_decay)
    e = torch.exp(log_decay.view(-1, *[1] * d.dim()) * d.clamp_min(0))
    return torch.where(d >= 0, e, 0.0)


def _scan(a, b, c, log_decay, first, late):
    """out_i = sum over j <= i of d^(i - j) (a_i . b_j) c_j + d^(i + 1 - late) a_i . first, and the last state, sum over j of
    d^(T - 1 + late - j) b_j c_j^T + d^T first; of [batch, heads, T, .] operands, chunk by chunk. The batch's sequences may have fewer
    than T rows: those behind them are zeros, and the caller scales."""
    tokens = a.shape[2]
    a, b, c = (torch.nn.functional.pad(t, (0, 0, 0, -tokens % CHUNK)).unflatten(2, (-1, CHUNK)) for t in (a, b, c))
    at = torch.arange(CHUNK, device=a.device)
    order = torch.arange(a.shape[2], device=a.device)
    inner = (a @ b.transpose(-1, -2)) * _decay(log_decay, at[:, None] - at)[:, None] @ c
    added = (b * _decay(log_decay, CHUNK - 1 + late - at)[:, None, :, None]).transpose(-1, -2) @ c
    before = _decay(log_decay, CHUNK * (order[:, None] - order - 1)) @ added.flatten(3)
    before = before + _decay(log_decay, CHUNK * order)[..., None] * first.flatten(2).unsqueeze(2)
    outer = (a * _decay(log_decay, at + 1 - late)[:, None, :, None]) @ before.unflatten(3, first.shape[2:])
    return (inner + outer).flatten(2, 3)[:, :, :tokens]


def _last(b, c, log_decay, first, late, lengths):
    """The state behind each sequence's last row: sum over j of d^(length - 1 + late - j) b_j c_j^T + d^length first."""
    left = lengths[:, None] - 1 + late - torch.arange(b.shape[2], device=b.device)
    w = _decay(log_decay, torch.where(left >= late, left, -1)).transpose(0, 1)
    return (b * w.unsqueeze(-1)).transpose(-1, -2) @ c + _decay(log_decay, lengths).t()[..., None, None] * first


def _by_sequence(s, t, heads):
    """[.., heads, dim] as float32 [batch, heads, T, dim] with the shared heads repeated, rows behind a sequence's end zero."""
    t = t.float()
    if "offsets" in s:
        o = s["offsets"].long()
        at = o[:-1, None] + torch.arange(s["most"], device=t.device)
        t = torch.where((at < o[1:, None])[..., None, None], t[at.clamp_max(t.shape[0] - 1)], 0.0)
    return t.transpose(1, 2).repeat_interleave(heads // t.shape[-2], 1)


def _back(s, t, kv_heads):
    """The inverse: summed over the heads that share, in the operands' layout and type."""
    t = t.unflatten(1, (kv_heads, -1)).sum(2).transpose(1, 2)
    if "offsets" in s:
        o = s["offsets"].long()
        row = torch.arange(s["q"].shape[0], device=t.device)
        which = torch.searchsorted(o[1:], row, right=True)
        t = t[which, row - o[which]]
    return t.to(s["dtype"])


def _turned(s, t, lengths):
    """Each sequence's rows from its last to its first."""
    at = (lengths[:, None] - 1 - torch.arange(t.shape[2], device=t.device)).view(t.shape[0], 1, -1, 1)
    return torch.where(at >= 0, torch.take_along_dim(t, at.clamp_min(0), 2), 0.0)


def _plain_attention(s):
    s = dict(s)
    heads, dim, kv_heads = *s["q"].shape[-2:], s["k"].shape[-2]
    if "offsets" in s:
        lengths = s["offsets"].long().diff()
        s["most"] = int(lengths.max())
    else:
        lengths = torch.full((s["q"].shape[0],), s["q"].shape[1], device=s["q"].device)
    q, k, v = (_by_sequence(s, s[name], heads) for name in ("q", "k", "v"))
    g, scale = s["log_decay"], 1 / math.sqrt(dim)
    first = s["state"] if "state" in s else q.new_zeros(q.shape[0], heads, dim, v.shape[-1])
    got = {"out": _back(s, scale * _scan(q, k, v, g, first, 0), heads), "state": _last(k, v, g, first, 0, lengths)}
    if "go" not in s:
        return got
    go = _by_sequence(s, s["go"], heads)
    last = s["gs"] if "gs" in s else torch.zeros_like(first)
    got["gq"] = _back(s, scale * _scan(go, v, k, g, first.transpose(-1, -2), 0), heads)
    q = scale * q
    if "gs" in s:
        got["gs"] = _last(_turned(s, q, lengths), _turned(s, go, lengths), g, last, 1, lengths)
    q, k, v, go = (_turned(s, t, lengths) for t in (q, k, v, go))
    got["gk"] = _back(s, _turned(s, _scan(v, go, q, g, last.transpose(-1, -2), 1), lengths), kv_heads)
    got["gv"] = _back(s, _turned(s, _scan(k, q, go, g, last, 1), lengths), kv_heads)
    return got


def _plain_step(s):
    state, heads, dim = s["state"], *s["q"].shape[-2:]
    q, k, v = (s[name].float().repeat_interleave(heads // s[name].shape[1], 1) for name in ("q", "k", "v"))
    now = torch.exp(s["log_decay"])[:, None, None] * (state if s["slots"] is None else state[s["slots"]]) + k.unsqueeze(-1) * v.unsqueeze(-2)
    if s["slots"] is None:
        state.copy_(now)
    else:
        state[s["slots"]] = now
    return {"out": (q.unsqueeze(-2) @ now).squeeze(-2).mul(1 / math.sqrt(dim)).to(s["dtype"]), "state": state}


def _plain(s):
    if s["op"] == "rotary_train":
        cos, sin = _angles(s)
        y = _rotated(s["x"].float(), cos, sin, s["interleaved"]).to(s["dtype"])
        return {"y": y, "gx": _rotated(s["gy"].float(), cos, -sin, s["interleaved"]).to(s["dtype"])}
    if s["op"].startswith("norm"):
        return _plain_norm_rotary(s)
    return _plain_step(s) if s["op"] == "step" else _plain_attention(s)


# The framework's operators.


def _own(s):
    import morphocore_amd.functional as F

    op = s["op"]
    if op == "rotary_train":
        y = F.axial_rotary(s["x"], s["positions"], s["frequencies"], interleaved=s["interleaved"])
        return {"y": y, "gx": torch.autograd.grad(y, s["x"], s["gy"])[0]}
    if op == "norm_rotary_infer":
        with torch.no_grad():
            q, k = F.rms_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["frequencies"], eps=EPS, interleaved=s["interleaved"])
        return {"q": q, "k": k}
    if op == "norm_rotary_train":
        q, k = F.rms_norm_rotary(s["q"], s["k"], s["qw"], s["kw"], s["positions"], s["frequencies"], eps=EPS, interleaved=s["interleaved"])
        gq, gk, gqw, gkw = torch.autograd.grad([q, k], [s["q"], s["k"], s["qw"], s["kw"]], [s["gq"], s["gk"]])
        return {"q": q, "k": k, "gq": gq, "gk": gk, "gqw": gqw, "gkw": gkw}
    if op == "step":
        with torch.no_grad():
            return {"out": F.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"]), "state": s["state"]}
    if op == "attention":
        with torch.no_grad():
            out, last = F.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], offsets=s.get("offsets"), final_state=True)
        return {"out": out, "state": last}
    out, last = F.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s.get("state"), offsets=s.get("offsets"), final_state=True)
    got = {"out": out.detach(), "state": last.detach()}
    if "gs" in s:
        got["gq"], got["gk"], got["gv"], got["gs"] = torch.autograd.grad([out, last], [s["q"], s["k"], s["v"], s["state"]], [s["go"], s["gs"]])
    else:
        got["gq"], got["gk"], got["gv"] = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["go"])
    return got


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    """Bytes: inputs and outputs once. Flops: a handful a value of norm and rotation; of attention the products with each token's
    state, forward 2 (the update, the output), backward 5 (the state again, its gradient's update, the three gradients)."""
    size, op, dim = SIZE[case["dtype"]], case["op"], case["dim"]
    if op == "rotary_train":
        n = case["batch"] * case["frames"] * case["height"] * case["width"] * case["heads"] * dim
        return {"bytes": 4 * n * size, "flops": 6 * n}
    if op.startswith("norm"):
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * dim
        return {"bytes": n * size * (5 if op.endswith("train") else 2), "flops": (22 if op.endswith("train") else 8) * n}
    heads, kv_heads, value_dim, batch = case["heads"], case["kv_heads"], case["value_dim"], case["batch"]
    product, states = heads * dim * value_dim, batch * heads * dim * value_dim * 4
    if op == "step":
        rows = batch
        return {"bytes": 2 * states + rows * size * (heads * (dim + value_dim) + kv_heads * (dim + value_dim)), "flops": 5 * rows * product}
    rows = case["tokens"] * (1 if case["ragged"] else batch)
    read, written = rows * size * (heads * dim + kv_heads * (dim + value_dim)), rows * size * heads * value_dim
    if op == "attention":
        return {"bytes": read + written + states, "flops": 4 * rows * product}
    return {"bytes": 2 * read + 2 * written + states * (4 if case["ragged"] else 1), "flops": 14 * rows * product}


# The definition in 64 bits.


def _exact_turn(s, x, sign):
    """Pair by pair as complex numbers."""
    angle = (s["positions"].double().unsqueeze(-1) * s["frequencies"]).sum(-2)
    pairs = angle.shape[-1]
    unit = torch.polar(torch.ones_like(angle), sign * angle).unsqueeze(-2)
    y = x.clone()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if s["interleaved"] else (slice(0, pairs), slice(pairs, 2 * pairs))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_sequence(q, k, v, g, first, go, last, scale):
    """One head of one sequence by every pair of tokens, a block of rows at a time."""
    n, block = q.shape[0], 1024
    at = torch.arange(n, device=q.device, dtype=torch.float64)
    far = torch.exp(g * (at + 1)).unsqueeze(1)
    near = torch.exp(g * (n - 1 - at)).unsqueeze(1)
    out = torch.empty(n, v.shape[1], dtype=torch.float64, device=q.device)
    gq, gk, gv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(0, n, block):
        rows = slice(i, min(n, i + block))
        seen = slice(0, min(n, i + block))
        gap = at[rows].unsqueeze(1) - at[seen]
        weight = torch.exp(g * gap.clamp_min(0)) * (gap >= 0) * scale
        score = (q[rows] @ k[seen].t()) * weight
        out[rows] = score @ v[seen] + scale * far[rows] * (q[rows] @ first)
        if go is not None:
            gscore = (go[rows] @ v[seen].t()) * weight
            gq[rows] = gscore @ k[seen] + scale * far[rows] * (go[rows] @ first.t())
            gk[seen] += gscore.t() @ q[rows]
            gv[seen] += score.t() @ go[rows]
    final = (near * k).t() @ v + torch.exp(g * n) * first
    if go is None:
        return out, final, None, None, None, None
    return out, final, gq, gk + near * (v @ last.t()), gv + near * (k @ last), torch.exp(g * n) * last + scale * (far * q).t() @ go


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], {name: t.detach().double() for name, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if op == "rotary_train":
        return {"y": _exact_turn(s, d["x"], 1), "gx": _exact_turn(s, d["gy"], -1)}
    if op.startswith("norm"):
        got = {}
        for name in ("q", "k"):
            x, w = d[name], d[name + "w"]
            r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
            got[name] = _exact_turn(s, x * r * w, 1)
            if op.endswith("train"):
                g = _exact_turn(s, d["g" + name], -1)
                t = g * w
                got["g" + name] = r * t - x * r**3 * (t * x).mean(-1, keepdim=True)
                got["g" + name + "w"] = (g * x * r).sum((0, 1))
        return got
    heads, kv_heads = case["heads"], case["kv_heads"]
    scale, group = 1 / math.sqrt(case["dim"]), heads // kv_heads
    if op == "step":
        kept = d["state"]
        where = torch.arange(case["batch"], device=kept.device) if s["slots"] is None else s["slots"].long()
        out = torch.empty(case["batch"], heads, case["value_dim"], dtype=torch.float64, device=kept.device)
        for h in range(heads):
            kept[where, h] = torch.exp(d["log_decay"][h]) * kept[where, h] + torch.einsum("bi,bj->bij", d["k"][:, h // group], d["v"][:, h // group])
            out[:, h] = scale * (d["q"][:, h].unsqueeze(-1) * kept[where, h]).sum(1)
        return {"out": out, "state": kept}
    batch = case["batch"]
    if case["tokens"] * heads * batch * (1 if case["ragged"] else case["tokens"] / 4096) > 2**31 or batch * heads > 1024:
        return None
    offsets = s["offsets"].tolist() if case["ragged"] else [b * case["tokens"] for b in range(batch + 1)]
    q, k, v = (d[name].reshape(-1, *d[name].shape[-2:]) for name in ("q", "k", "v"))
    go = d["go"].reshape(-1, heads, case["value_dim"]) if "go" in d else None
    first = d["state"] if "state" in d else torch.zeros(batch, heads, case["dim"], case["value_dim"], dtype=torch.float64, device=q.device)
    last = d["gs"] if "gs" in d else torch.zeros_like(first)
    out, final = torch.zeros(q.shape[0], heads, case["value_dim"], dtype=torch.float64, device=q.device), torch.empty_like(first)
    gq, gk, gv, gs = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.empty_like(first)
    for b in range(batch):
        rows = slice(offsets[b], offsets[b + 1])
        for h in range(heads):
            o, f, a, c, e, r = _exact_sequence(q[rows, h], k[rows, h // group], v[rows, h // group], d["log_decay"][h], first[b, h],
                                               None if go is None else go[rows, h], last[b, h], scale)
            out[rows, h], final[b, h] = o, f
            if go is not None:
                gq[rows, h], gs[b, h] = a, r
                gk[rows, h // group] += c
                gv[rows, h // group] += e
    got = {"out": out.view(*s["q"].shape[:-1], -1), "state": final}
    if go is not None:
        got.update(gq=gq.view(s["q"].shape), gk=gk.view(s["k"].shape), gv=gv.view(s["v"].shape))
        if "gs" in d:
            got["gs"] = gs
    return got
