"""GPU parity of the 8-bit codes of ud_i8_quantize and ud_rms_norm at the borders between two of them: a code is the fp32 quotient
y / scale, rounded to the nearest whole number, the even one of two."""
import numpy as np
import pytest

from test_gpu_rows import norm, quantize

pytestmark = pytest.mark.gpu

f32 = np.float32


def at_borders(rng, rows):
    """fp32 rows [rows, 768] (of any magnitude) of the values next to the borders n + 1/2 of their own scale, and the codes."""
    top = (np.exp2(rng.uniform(-100, 100, rows)) * rng.uniform(1, 2, rows)).astype(f32)
    scale = top / f32(127)
    y = np.zeros((rows, 768), f32)
    y[:, 0] = top
    at = ((np.arange(127) + 0.5) * scale[:, None].astype(np.float64)).astype(f32)
    for i, v in enumerate((at, np.nextafter(at, f32(0)), np.nextafter(at, f32(np.inf)))):
        y[:, 1 + 254 * i:1 + 254 * i + 127] = v
        y[:, 1 + 254 * i + 127:1 + 254 * i + 254] = -v
    y = np.clip(y, -top[:, None], top[:, None])
    return y, scale, np.rint(y / scale[:, None]).astype(np.int8)


@pytest.mark.parametrize("pad", [0, 2, 3000])
def test_codes_at_borders(gpu, pad):
    """Rows of one wave and of several, whose values a product with the scale's reciprocal would give to the other code thousands of times."""
    y, scale, codes = at_borders(np.random.default_rng(1), 64)
    assert (np.rint(y * (f32(1) / scale)[:, None]) != codes).sum() > 4000
    wide = np.zeros((64, 768 + 8 * pad), f32)
    wide[:, -768:] = y
    got, scales = quantize(gpu, wide.astype(np.float64), None, "f32")
    np.testing.assert_array_equal(scales, scale.astype(np.float64))
    np.testing.assert_array_equal(got[:, -768:], codes)
    assert not got[:, :-768].any()


def test_norm_codes_at_borders(gpu):
    """eps of 1e30 beside squares of 1e10: the norm's factor does not hang on the order of their sum, and two products in fp32 follow."""
    rng = np.random.default_rng(2)
    y = (rng.standard_normal((40, 1024)) * 1e5).astype(f32)
    w = np.full(1024, 2.0 ** 50, f32)
    got, scales, _ = norm(gpu, y.astype(np.float64), None, w, "f32", "f32", True, eps=1e30)
    r = (1 / np.sqrt(np.mean(y.astype(np.float64) ** 2, 1) + float(f32(1e30)))).astype(f32)
    z = (y * r[:, None]) * w
    scale = np.abs(z).max(1) / f32(127)
    np.testing.assert_array_equal(scales, scale.astype(np.float64))
    np.testing.assert_array_equal(got, np.rint(z / scale[:, None]).astype(np.int8))
