"""The channel-mixing operators in numpy float64, from their definitions: 8-bit blocks (OCP E4M3 codes with
a power-of-two scale for 32 values), root-mean-square norm, gated activation, weight gradient."""
import numpy as np

BLOCK = 32


def e4m3_values():
    """The value of every code: sign, 4 exponent bits (bias 7), 3 significand bits; 0x7f / 0xff are NaN."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        mag = np.nan if (c & 0x7F) == 0x7F else (m / 8 * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        v[c] = -mag if c & 0x80 else mag
    return v


VALUES = e4m3_values()
_POSITIVE = VALUES[:0x7F]  # ascending


def encode(t):
    """Codes of t by nearest value, ties to the even code, saturated; NaN and infinities the NaN code."""
    a = np.abs(np.where(np.isfinite(t), t, 0.0))
    hi = np.clip(np.searchsorted(_POSITIVE, a), 1, len(_POSITIVE) - 1)
    lo = hi - 1
    mid = (_POSITIVE[lo] + _POSITIVE[hi]) / 2  # exact
    up = (a > mid) | ((a == mid) & (hi % 2 == 0))
    code = np.where(up, hi, lo).astype(np.uint8)
    code = np.where(np.signbit(t), code | 0x80, code)
    return np.where(np.isfinite(t), code, 0x7F).astype(np.uint8)


def pack(x):
    """(codes, scale bytes) of float64 values that are exact in float32."""
    cols = x.shape[-1]
    nb = -(-cols // BLOCK)
    v = np.zeros(x.shape[:-1] + (nb * BLOCK,))
    v[..., :cols] = x
    v = v.reshape(x.shape[:-1] + (nb, BLOCK))
    big = np.max(np.where(np.isfinite(v), np.abs(v), 0.0), axis=-1)
    e = np.full(big.shape, -117)
    for i in np.ndindex(big.shape):  # the smallest exponent by trial, independent of any bit pattern
        while e[i] < 119 and big[i] > 448 * 2.0 ** int(e[i]):
            e[i] += 1
    codes = encode(v / np.exp2(e.astype(np.float64))[..., None])
    return codes.reshape(x.shape[:-1] + (nb * BLOCK,))[..., :cols], (e + 127).astype(np.uint8)


def unpack(codes, scales):
    s = np.exp2(scales.astype(np.float64) - 127).repeat(BLOCK, axis=-1)[..., : codes.shape[-1]]
    return VALUES[codes] * s


def rms_norm(h, w, eps):
    return h / np.sqrt(np.mean(h * h, axis=-1, keepdims=True) + eps) * w


def rms_norm_grads(h, w, eps, gy, gh=0.0):
    """(grad of h as an input, grad of w); each with the sum of its terms' magnitudes, which scales its error."""
    r = 1 / np.sqrt(np.mean(h * h, axis=-1, keepdims=True) + eps)
    n, a = h * r, gy * w
    m = np.mean(a * n, axis=-1, keepdims=True)
    gx = r * (a - n * m) + gh
    size = r * (np.abs(a) + np.abs(n) * np.mean(np.abs(a * n), axis=-1, keepdims=True)) + np.abs(gh)
    lead = tuple(range(h.ndim - 1))
    return gx, (gy * n).sum(lead), size, np.abs(gy * n).sum(lead)


def sigmoid(g):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g))


def gated(g, u):
    return g * sigmoid(g) * u


def gated_grads(g, u, gy):
    s = sigmoid(g)
    return gy * u * s * (1 + g * (1 - s)), gy * g * s, np.abs(gy * u * s) * (1 + np.abs(g))
