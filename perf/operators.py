"""Cases of the channel-mixing operators: root-mean-square norm, 8-bit checkpoints, gated activation and
the weight gradient that reads a checkpoint.

Every case is one call as a program makes it: a training step's forward and backward (outputs and
gradients), or an inference forward. With ``own`` false, ``run`` computes the operators in elementary
torch operations in float32; with ``own`` true, through ``morphocore_amd.functional``.

8-bit blocks: 32 values of a row share the scale 2^e, e the smallest integer in [-117, 119] with
max |v| <= 448 * 2^e; a value is held as e4m3(v / 2^e). What is held in 8 bits is returned as the values
it stands for, which bfloat16 holds exactly.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
BLOCK = 32


def listed():
    return [
        # One token of a served model: the residual's addition, the norm and its 8-bit output, where only
        # the call's latency counts.
        dict(name="norm8_one_token", op="norm8_infer", dtype="bf16", rows=1, cols=4096),
        # A training step of a wide block's norm, whose 8-bit output is kept for the next layer's weight gradient.
        dict(name="norm8_train", op="norm8_train", dtype="bf16", rows=8192, cols=4096),
        # The pixels of the benchmark's image batch (8x64x256x256) with their 64 channels last, in float32.
        dict(name="norm_image_train", op="norm_train", dtype="f32", rows=524288, cols=64),
        # A ragged batch of a width that no vector divides, in float16.
        dict(name="norm8_odd_train", op="norm8_train", dtype="f16", rows=1531, cols=1237),
        # The checkpoint of a large activation, written and read back.
        dict(name="pack8_large", op="pack8", dtype="bf16", rows=16384, cols=8192),
        # A small checkpoint whose rows end inside a block.
        dict(name="pack8_odd", op="pack8", dtype="f32", rows=257, cols=1021),
        # The gated activation of a wide block in training, both halves of one projection.
        dict(name="gated8_train", op="gated8_train", dtype="bf16", rows=8192, cols=8192),
        # The same for a short batch of a narrow block: launches and host time.
        dict(name="gated8_small_train", op="gated8_train", dtype="f32", rows=64, cols=256),
        # An odd hidden width in float16.
        dict(name="gated8_odd_train", op="gated8_train", dtype="f16", rows=1999, cols=2731),
        # The weight gradient of a wide square layer: one large product.
        dict(name="weight_large", op="weight", dtype="bf16", rows=8192, out=4096, cols=4096),
        # The weight gradient of a layer over the benchmark's pixels: few channels, a very long sum.
        dict(name="weight_image", op="weight", dtype="f32", rows=524288, out=64, cols=64),
        # A weight gradient of which no side is a multiple of a tile.
        dict(name="weight_odd", op="weight", dtype="f16", rows=5003, out=1111, cols=777),
    ]


def _log(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    n += rng.random() < 0.5 and n % 2 == 0 and low < n < high
    return n + (n == 3072)


def draw(rng):
    op = rng.choice(["norm8_infer", "norm8_train", "norm_train", "pack8", "gated8_train", "weight", "weight"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    while True:
        rows, cols = _log(rng, 1, 524288), _log(rng, 16, 12288)
        case = dict(op=op, dtype=dtype, rows=rows, cols=cols)
        if op == "weight":
            case["out"] = _log(rng, 16, 12288)
            if rows * cols * case["out"] <= 2**37 and rows * max(cols, case["out"]) <= 2**26 and case["out"] * cols <= 2**26:
                return case
        elif op == "norm8_infer" and rows > 64:
            continue
        elif rows * cols <= 2**25:
            return case


def _row_scale(g, rows):
    """The spread of a batch's rows: some are several times others."""
    return torch.exp(0.5 * torch.randn(rows, 1, generator=g, device="cuda"))


def _activations(g, rows, cols, dtype, above=20.0):
    """Activations: rows of several sizes, a few channels far above the others (as in a residual stream)."""
    x = torch.randn(rows, cols, generator=g, device="cuda") * _row_scale(g, rows)
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(loud, above * x, x).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype, rows, cols = case["op"], DTYPES[case["dtype"]], case["rows"], case["cols"]
    train = op.endswith("_train")

    def gradient(*shape):
        return (torch.randn(shape, generator=g, device="cuda") * 0.05).to(dtype)

    state = {"op": op, "dtype": dtype}
    if op.startswith("norm"):
        state["x"] = _activations(g, rows, cols, dtype).requires_grad_(train)
        state["weight"] = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype).requires_grad_(train)
        if op.startswith("norm8"):
            state["residual"] = _activations(g, rows, cols, dtype).requires_grad_(train)
        if train:
            state["gy"] = gradient(rows, cols)
            if op == "norm8_train":
                state["gh"] = gradient(rows, cols)
    elif op == "pack8":
        state["x"] = _activations(g, rows, cols, dtype)
    elif op == "gated8_train":
        state["x"] = _activations(g, rows, 2 * cols, dtype, above=5.0).requires_grad_(True)
        state["gy"] = gradient(rows, cols)
    else:
        state["gy"] = gradient(rows, case["out"])
        state["codes"], state["scales"] = _pack(_activations(g, rows, cols, torch.bfloat16))
    return state


# The plain form.


def _power_of_two(e):
    return ((e + 127) << 23).view(torch.float32)


def _blocks(v):
    return torch.nn.functional.pad(v, (0, -v.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))


def _pack(x):
    """The codes (float8_e4m3fn, of x's shape) and scales (float8_e8m0fnu, one a block) of x's 8-bit form."""
    v = _blocks(x.float())
    finite = torch.isfinite(v)
    largest = torch.where(finite, v.abs(), 0.0).amax(-1)
    m, k = torch.frexp(largest)
    e = torch.where(largest > 0, k - 9 + (m > 0.875).to(torch.int32), -117).clamp(-117, 119)
    q = (v * _power_of_two(-e).unsqueeze(-1)).clamp(-448.0, 448.0)
    codes = torch.where(finite, q, math.nan).to(torch.float8_e4m3fn)
    return codes.flatten(-2)[..., : x.shape[-1]].contiguous(), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _unpack(codes, scales):
    """The values in float32."""
    cols = codes.shape[-1]
    scale = _power_of_two(scales.view(torch.uint8).to(torch.int32) - 127)
    return (_blocks(codes.float()) * scale.unsqueeze(-1)).flatten(-2)[..., :cols]


def _plain_norm(s):
    dtype, h, w = s["dtype"], s["x"].float(), s["weight"].float()
    if "residual" in s:
        h = h + s["residual"].float()
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    n = h * rstd
    y = (n * w).to(dtype)
    got = {}
    if s["op"].startswith("norm8"):
        got["packed"] = _unpack(*_pack(y)).to(torch.bfloat16)
        got["h"] = h.to(dtype)
    if s["op"] == "norm8_infer":
        return got
    gy = s["gy"].float()
    gn = gy * w
    gx = rstd * (gn - n * (gn * n).mean(-1, keepdim=True))
    if "gh" in s:
        gx = gx + s["gh"].float()
        got["gr"] = gx.to(dtype)
    return {**got, "y": y, "gx": gx.to(dtype), "gw": (gy * n).sum(0).to(dtype)}


def _plain_gated(s):
    dtype, x, gy = s["dtype"], s["x"].float(), s["gy"].float()
    g, u = x.chunk(2, -1)
    y = (g / (1 + torch.exp(-g)) * u).to(dtype)
    g, u = _unpack(*_pack(g)), _unpack(*_pack(u))
    sg = 1 / (1 + torch.exp(-g))
    gx = torch.cat([gy * u * sg * (1 + g * (1 - sg)), gy * g * sg], -1)
    return {"y": y, "packed": _unpack(*_pack(y)).to(torch.bfloat16), "gx": gx.to(dtype)}


def _plain(s):
    if s["op"].startswith("norm"):
        return _plain_norm(s)
    if s["op"] == "pack8":
        return _unpack(*_pack(s["x"])).to(torch.bfloat16)
    if s["op"] == "gated8_train":
        return _plain_gated(s)
    return (s["gy"].float().t() @ _unpack(s["codes"], s["scales"])).to(s["dtype"])


# The framework's operators.


def _own(s):
    import morphocore_amd.functional as F

    op, x = s["op"], s.get("x")
    if op == "norm8_infer":
        with torch.no_grad():
            _, packed, h = F.rms_norm8(x, s["weight"], s["residual"], EPS, full=False)
            return {"packed": F.unpack8(packed, torch.bfloat16), "h": h}
    if op == "norm8_train":
        y, packed, h = F.rms_norm8(x, s["weight"], s["residual"], EPS)
        gx, gr, gw = torch.autograd.grad([y, h], [x, s["residual"], s["weight"]], [s["gy"], s["gh"]])
        return {"packed": F.unpack8(packed, torch.bfloat16), "h": h, "y": y, "gx": gx, "gr": gr, "gw": gw}
    if op == "norm_train":
        y = F.rms_norm(x, s["weight"], eps=EPS)
        gx, gw = torch.autograd.grad(y, [x, s["weight"]], s["gy"])
        return {"y": y, "gx": gx, "gw": gw}
    if op == "pack8":
        return F.unpack8(F.pack8(x), torch.bfloat16)
    if op == "gated8_train":
        y, packed = F.gated_silu8(x)
        (gx,) = torch.autograd.grad(y, [x], s["gy"])
        return {"y": y, "packed": F.unpack8(packed, torch.bfloat16), "gx": gx}
    return F.grad_weight8(s["gy"], F.Packed8(s["codes"], s["scales"]))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    """Bytes: inputs and outputs once. Flops: of the elementwise operators a handful a value, of the weight
    gradient's product a multiplication and an addition a term."""
    size, rows, cols = SIZE[case["dtype"]], case["rows"], case["cols"]
    n, op = rows * cols, case["op"]
    if op == "norm8_infer":  # x, r; values of the codes, h
        return {"bytes": n * (3 * size + 2) + cols * size, "flops": 8 * n}
    if op == "norm8_train":  # x, r, gy, gh; y, values of the codes, h, gx, gr
        return {"bytes": n * (9 * size + 2) + 2 * cols * size, "flops": 20 * n}
    if op == "norm_train":  # x, gy; y, gx
        return {"bytes": n * 4 * size + 2 * cols * size, "flops": 16 * n}
    if op == "pack8":
        return {"bytes": n * (size + 2), "flops": 3 * n}
    if op == "gated8_train":  # x, gy; y, values of the codes, gx
        return {"bytes": n * (6 * size + 2), "flops": 30 * n}
    out = case["out"]
    return {"bytes": rows * out * size + n + rows * -(-cols // BLOCK) + out * cols * size, "flops": 2 * n * out}


# The definition in 64 bits.


def _exact_held(v):
    """The values that 8-bit blocks hold of v (float64)."""
    rows, cols = v.shape
    blocks = -(-cols // BLOCK)
    held = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64, device=v.device)
    held[:, :cols] = v
    held = held.view(rows, blocks, BLOCK)
    ratio = held.abs().amax(2, keepdim=True) / 448
    scale = torch.exp2(torch.ceil(torch.log2(ratio.clamp_min(2.0**-117))))
    t = held / scale
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0**-6))) - 3)
    return (torch.round(t / step) * step * scale).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.dtype in DTYPES.values()}
    op = case["op"]
    if op.startswith("norm"):
        h = d["x"] + d["residual"] if "residual" in d else d["x"]
        r = 1 / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
        y = h * r * d["weight"]
        got = {}
        if op.startswith("norm8"):
            got = {"packed": _exact_held(y.to(s["dtype"]).double()), "h": h}
        if op == "norm8_infer":
            return got
        t = d["gy"] * d["weight"]
        gx = r * t - h * r**3 * (t * h).mean(1, keepdim=True)
        if "gh" in d:
            gx = gx + d["gh"]
            got["gr"] = gx
        return {**got, "y": y, "gx": gx, "gw": (d["gy"] * h * r).sum(0)}
    if op == "pack8":
        return _exact_held(d["x"])
    if op == "gated8_train":
        half = case["cols"]
        g, u = d["x"][:, :half], d["x"][:, half:]
        y = g * u * torch.sigmoid(g)
        g, u = _exact_held(g), _exact_held(u)
        sg = torch.sigmoid(g)
        gx = torch.empty_like(d["x"])
        gx[:, half:] = d["gy"] * g * sg
        gx[:, :half] = d["gy"] * u * (sg + g * sg * (1 - sg))
        return {"y": y, "packed": _exact_held(y.to(s["dtype"]).double()), "gx": gx}
    scale = torch.exp2(s["scales"].view(torch.uint8).double() - 127).repeat_interleave(BLOCK, 1)[:, : case["cols"]]
    held = s["codes"].float().double() * scale
    return torch.mm(d["gy"].t(), held)
