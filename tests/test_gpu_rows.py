"""GPU parity of ud_rms_norm and ud_i8_quantize with their float64 forms (layer_ref.py): every type, every kernel shape
(dims of 8 to 32768), strided rows, in place, far values, rows that are no numbers."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu

EPS = 1e-6
# s * r * w: the rounding of r, and three products' (r's square root and division are in 64 bits)
NORM_REL = 4 * ref.STEP32
# exp off by 2^-23 of its value and v_rcp by 2^-23, 1 + e, x * g and the product: 8 half steps; one to spare
GATE_REL = 9 * ref.STEP32


def dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def padded(bits, ld, fill):
    out = np.full((len(bits), ld), fill, bits.dtype)
    out[:, :bits.shape[1]] = bits
    return out


def norm(ud, x, res, weight, dtype, sum_dtype, eight, ld=0, in_place=False, eps=EPS):
    """x, res: float64 values of their types.  (out bits or codes, scales, sum bits); checks what lies behind the rows."""
    rows, dim = x.shape
    ld = dim + ld
    xb, _ = ref.stored(x, dtype)
    xd = dev(ud, padded(xb, ld, 3))
    wd = dev(ud, weight) if weight is not None else None
    rd = sd = None
    if res is not None:
        rb, _ = ref.stored(res, sum_dtype)
        rd = dev(ud, padded(rb, ld, 5))
        sd = rd if in_place else dev(ud, np.full((rows, ld), 5, rb.dtype))
    if eight:
        od, scd = dev(ud, np.full((rows, ld), 77, np.int8)), dev(ud, np.full(rows + 1, 9, np.float32))
    else:
        od, scd = (xd, None) if in_place else (dev(ud, np.full((rows, ld), 3, xb.dtype)), None)
    ud.rms_norm(xd, od, rows, dim, weight=wd, eps=eps, residual=rd, sum_out=sd, scales=scd, dtype=dtype, sum_dtype=sum_dtype,
                out_dtype="i8" if eight else None, x_ld=ld, sum_ld=ld, out_ld=ld)
    ud.synchronize()
    out = od.download((rows, ld), np.int8 if eight else xb.dtype)
    assert np.all(out[:, dim:] == (77 if eight else 3))
    scales = sums = None
    if eight:
        scales = scd.download(rows + 1)
        assert scales[-1] == 9
        scales = scales[:-1].astype(np.float64)
    if res is not None:
        sums = sd.download((rows, ld), rb.dtype)
        assert np.all(sums[:, dim:] == 5)
        sums = sums[:, :dim]
    return out[:, :dim], scales, sums


def check_norm(ud, rng, rows, dim, dtype, sum_dtype, eight, residual=True, weight=True, ld=0, in_place=False, scale=1.0):
    x = ref.stored(scale * rng.standard_normal((rows, dim)) * np.exp(rng.standard_normal((1, dim))), dtype)[1]
    res = ref.stored(4 * scale * rng.standard_normal((rows, dim)), sum_dtype)[1] if residual else None
    w = (1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if weight else None
    out, scales, sums = norm(ud, x, res, w, dtype, sum_dtype, eight, ld, in_place)
    s = ref.summed(x, res, sum_dtype)
    if residual:
        np.testing.assert_array_equal(ref.from_bits(sums, sum_dtype), s)
    y = ref.normed(s, w, EPS)
    if eight:
        ref.check_codes(out, scales, y, NORM_REL)
    else:
        got = ref.from_bits(out, dtype)
        assert np.all(np.abs(got - y) <= (ref.HALF_STEP[dtype] * 1.01 + NORM_REL) * np.abs(y) + ref.FLOOR[dtype])


TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f32", "f32")]
DIMS = [8, 504, 512, 520, 1024, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16392, 32768]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype,sum_dtype", TYPES)
def test_norm_dims(gpu, dtype, sum_dtype, dim):
    rng = np.random.default_rng([dim, len(dtype), len(sum_dtype)])
    for rows in (1, 5):
        check_norm(gpu, rng, rows, dim, dtype, sum_dtype, False)
        check_norm(gpu, rng, rows, dim, dtype, sum_dtype, True, weight=rows == 1)
    check_norm(gpu, rng, 3, dim, dtype, sum_dtype, True, residual=False, ld=16)
    check_norm(gpu, rng, 3, dim, dtype, sum_dtype, False, in_place=True, ld=8)


@pytest.mark.parametrize("dim", [24, 1000, 1032, 2040, 2064, 4000, 6008])
@pytest.mark.parametrize("dtype,sum_dtype", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
def test_norm_many_rows(gpu, dtype, sum_dtype, dim):
    rng = np.random.default_rng([dim, 7])
    check_norm(gpu, rng, 1027, dim, dtype, sum_dtype, True)
    check_norm(gpu, rng, 1025, dim, dtype, sum_dtype, False, in_place=True, ld=8)


def test_norm_far_values(gpu):
    """Rows whose squares are past fp32's range, or under it; zero rows."""
    rng = np.random.default_rng(3)
    check_norm(gpu, rng, 3, 640, "f32", "f32", False, scale=1e25)
    check_norm(gpu, rng, 3, 640, "bf16", "f32", True, scale=1e25)
    x = ref.stored(1e-25 * rng.standard_normal((2, 640)), "bf16")[1]
    for eight in (False, True):
        out, scales, _ = norm(gpu, x, None, None, "bf16", "bf16", eight, eps=1e-30)
        y = ref.normed(x, None, float(np.float32(1e-30)))
        if eight:
            ref.check_codes(out, scales, y, NORM_REL)
        else:
            assert np.all(np.abs(ref.from_bits(out, "bf16") - y) <= (2.0 ** -8 * 1.01 + NORM_REL) * np.abs(y))
    out, scales, _ = norm(gpu, np.zeros((2, 64)), np.zeros((2, 64)), None, "f16", "f32", True)
    assert np.all(out == 0) and np.all(scales == ref.TINY)


def test_norm_half_sums_saturate(gpu):
    x = np.full((1, 64), 60000.0)
    out, _, sums = norm(gpu, ref.stored(x, "f16")[1], ref.stored(x, "f16")[1], None, "f16", "f16", False)
    assert np.all(ref.from_bits(sums, "f16") == 65504) and np.all(ref.from_bits(out, "f16") == 1)


@pytest.mark.parametrize("dim", [256, 3000, 16000])
def test_rows_that_are_no_numbers(gpu, dim):
    rng = np.random.default_rng(dim)
    x = ref.stored(rng.standard_normal((6, dim)), "bf16")[1]
    clean = x.copy()
    x[1, dim - 1], x[3, 0], x[4, 5] = np.nan, np.inf, -np.inf
    for eight in (True, False):
        out, scales, _ = norm(gpu, x, None, None, "bf16", "bf16", eight)
        same, same_scales, _ = norm(gpu, clean, None, None, "bf16", "bf16", eight)
        np.testing.assert_array_equal(out[[0, 2, 5]], same[[0, 2, 5]])
        if eight:
            assert np.all(np.isnan(scales[[1, 3, 4]])) and np.all(out[[1, 3, 4]] == 0)
            np.testing.assert_array_equal(scales[[0, 2, 5]], same_scales[[0, 2, 5]])
        else:
            assert np.all(np.isnan(ref.from_bits(out, "bf16")[1]))
    codes, scales = quantize(gpu, x, None, "bf16")
    ref.check_codes(codes, scales, x, 0.0)


def quantize(ud, x, gate, dtype, fused=False, ld=0):
    rows, dim = x.shape
    xb = ref.stored(x, dtype)[0]
    gb = ref.stored(gate, dtype)[0] if gate is not None else None
    cd, sd = dev(ud, np.full((rows, dim + 16), 77, np.int8)), dev(ud, np.full(rows + 1, 9, np.float32))

    class At:
        def __init__(self, buf, off):
            self.buf, self.ptr = buf, buf.ptr + off

    if fused:
        both = dev(ud, padded(np.concatenate([gb, xb], 1), 2 * dim + ld, 3))
        gd, xd, dist = At(both, 0), At(both, dim * xb.itemsize), 2 * dim + ld
    else:
        xd, gd, dist = dev(ud, padded(xb, dim + ld, 3)), dev(ud, padded(gb, dim + ld, 3)) if gb is not None else None, dim + ld
    ud.i8_quantize(xd, cd, sd, rows, dim, gate=gd, dtype=dtype, ld=dist, codes_ld=dim + 16)
    ud.synchronize()
    c, s = cd.download((rows, dim + 16), np.int8), sd.download(rows + 1)
    assert np.all(c[:, dim:] == 77) and s[-1] == 9
    return c[:, :dim], s[:-1].astype(np.float64)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_dims(gpu, dtype, dim):
    rng = np.random.default_rng([dim, len(dtype)])
    for rows in (1, 5):
        x = ref.stored(rng.standard_normal((rows, dim)) * np.exp(rng.standard_normal((1, dim))), dtype)[1]
        g = ref.stored(3 * rng.standard_normal((rows, dim)), dtype)[1]
        ref.check_codes(*quantize(gpu, x, None, dtype, ld=8), x, 0.0)
        ref.check_codes(*quantize(gpu, x, g, dtype, fused=rows == 5, ld=8), ref.gated(x, g), GATE_REL)


@pytest.mark.parametrize("dim", [24, 1000, 2040, 4000, 6008])
def test_quantize_many_rows(gpu, dim):
    rng = np.random.default_rng([dim, 9])
    x = ref.stored(rng.standard_normal((1027, dim)), "bf16")[1]
    g = ref.stored(3 * rng.standard_normal((1027, dim)), "bf16")[1]
    ref.check_codes(*quantize(gpu, x, g, "bf16", fused=True), ref.gated(x, g), GATE_REL)
    ref.check_codes(*quantize(gpu, x, None, "bf16"), x, 0.0)


def test_quantize_borders_and_far_values(gpu):
    x = np.zeros((5, 64))
    x[0, :6] = [127, 0.5, 1.5, 2.5, -0.5, -3.5]            # scale 1: ties go to the even code
    x[1, :2] = [3e38, -3e38]
    x[2, :3] = [1e-40, -1e-40, 1e-38]                      # the scale stays normal: codes of multiples of 2^-126
    x[4, :2] = [-127 * 2.0 ** -126, 60 * 2.0 ** -126]
    codes, scales = quantize(gpu, x, None, "f32")
    assert list(codes[0, :6]) == [127, 0, 2, 2, 0, -4]
    assert list(codes[1, :2]) == [127, -127]
    assert list(codes[2, :3]) == [0, 0, 1] and scales[2] == ref.TINY
    assert np.all(codes[3] == 0) and scales[3] == ref.TINY
    assert list(codes[4, :2]) == [-127, 60]
    g = np.zeros((3, 64))
    g[0, :4] = [-60, -80, 80, 0]                           # far gates, a shut one, and one at infinity
    g[1, :2] = [-np.inf, 1]
    g[2, :2] = [np.inf, 1]
    y = np.ones((3, 64))
    codes, scales = quantize(gpu, y, g, "f32")
    ref.check_codes(codes[:1], scales[:1], ref.gated(y, g)[:1], GATE_REL)
    assert np.isnan(scales[2]) and np.all(codes[2] == 0)
    assert np.isnan(scales[1])                             # -inf / inf
    far = np.full((1, 64), -70.0)                          # all of a row at a far gate: relative to its own largest
    ref.check_codes(*quantize(gpu, np.arange(1, 65.0)[None], far + np.arange(64) / 64, "f32"),
                    ref.gated(np.arange(1, 65.0)[None], far + np.arange(64) / 64), GATE_REL)


def test_no_rows(gpu):
    b = dev(gpu, np.zeros(64, np.float32))
    gpu.rms_norm(b, b, 0, 8, dtype="f32")
    gpu.i8_quantize(b, b, b, 0, 8, dtype="f32")
