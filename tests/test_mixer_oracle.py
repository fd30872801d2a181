"""The channel-mixing oracle on the CPU: its 8-bit blocks against torch's conversions and against hand-made
values, its gradients against central differences of its own forward."""
import numpy as np
import pytest
import torch

from tests import mixer_oracle as O


def test_code_values_are_torch_float8():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.VALUES, want, equal_nan=True)


def test_encode_is_torch_rounding():
    x = np.concatenate([np.linspace(-448, 448, 30011), np.geomspace(2.0**-12, 448, 5000), O.VALUES[:0x7F],
                        (O.VALUES[:0x7E] + O.VALUES[1:0x7F]) / 2]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(O.encode(x.astype(np.float64)), want)


@pytest.mark.parametrize("cols", [1, 31, 32, 33, 100])
def test_pack_scale_is_the_smallest_that_holds_the_block(cols):
    rng = np.random.default_rng(cols)
    x = (rng.standard_normal((5, cols)) * np.exp(rng.standard_normal((5, 1)) * 8)).astype(np.float32).astype(np.float64)
    codes, scales = O.pack(x)
    for b in range(scales.shape[1]):
        big = np.abs(x[:, 32 * b: 32 * b + 32]).max(axis=1)
        e = scales[:, b].astype(int) - 127
        assert np.all(big <= 448 * 2.0**e) and np.all((big > 448 * 2.0 ** (e - 1)) | (e == -117))
    v = O.unpack(codes, scales)
    s = np.exp2(scales.astype(np.float64) - 127).repeat(32, axis=1)[:, :cols]
    assert np.all(np.abs(v - x) <= np.maximum(np.abs(x) / 16, s * 2.0**-10))


def test_special_blocks():
    x = np.zeros((1, 64))
    x[0, :4] = [np.inf, -np.inf, np.nan, 3.0]
    x[0, 40] = 3.4e38
    codes, scales = O.pack(x)
    v = O.unpack(codes, scales)
    assert np.isnan(v[0, :3]).all() and v[0, 3] == 3.0
    assert scales[0, 1] == 246 and v[0, 40] == 448 * 2.0**119
    assert O.pack(np.zeros((1, 32)))[1][0, 0] == 10


def _difference(f, x, d, step=1e-6):
    return (f(x + step * d) - f(x - step * d)) / (2 * step)


def test_gradients_are_the_forwards():
    rng = np.random.default_rng(0)
    h, w, gy, d = rng.standard_normal((3, 17)), 1 + rng.standard_normal(17) * 0.2, rng.standard_normal((3, 17)), rng.standard_normal((3, 17))
    gx, gw, _, _ = O.rms_norm_grads(h, w, 1e-6, gy)
    assert abs(_difference(lambda t: (O.rms_norm(t, w, 1e-6) * gy).sum(), h, d) - (gx * d).sum()) < 1e-7
    dw = rng.standard_normal(17)
    assert abs(_difference(lambda t: (O.rms_norm(h, t, 1e-6) * gy).sum(), w, dw) - (gw * dw).sum()) < 1e-7
    u = rng.standard_normal((3, 17))
    gg, gu, _ = O.gated_grads(h, u, gy)
    assert abs(_difference(lambda t: (O.gated(t, u) * gy).sum(), h, d) - (gg * d).sum()) < 1e-7
    assert abs(_difference(lambda t: (O.gated(h, t) * gy).sum(), u, d) - (gu * d).sum()) < 1e-7
