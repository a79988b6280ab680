"""GPU parity of ud_i8_linear with its float64 form (layer_ref.py): types, one row to many, odd sizes, strides, the largest
sums, bias and residual."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu


def dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


class At:
    def __init__(self, buf, off):
        self.buf, self.ptr = buf, buf.ptr + off


def run(ud, codes, scales, w, w_scales, dtype, bias=None, residual=None, pad=(0, 0, 0, 0), off=0, in_place=False):
    """pad: what the rows of codes, w, residual and out have behind them; off: elements that out and residual are off from
    the start of their buffers."""
    (M, K), N = codes.shape, len(w)

    def rows(a, ld, fill):
        out = np.full((len(a), ld), fill, a.dtype)
        out[:, :a.shape[1]] = a
        return dev(ud, out)

    cd, wd = rows(codes, K + pad[0], 99), rows(w, K + pad[1], 99)
    sd, wsd = dev(ud, scales.astype(np.float32)), dev(ud, w_scales.astype(np.float32))
    bd = dev(ud, bias.astype(np.float32)) if bias is not None else None
    kind = ref.to_bits(np.zeros(1), dtype).dtype
    old = N + pad[3]
    host = np.full(M * old + off + 8, 5, kind)
    rd, rld = None, N + pad[2]
    if residual is not None:
        rb = ref.stored(residual, dtype)[0]
        if in_place:
            rld = old
            host[off:off + M * old].reshape(M, old)[:, :N] = rb
        else:
            r = np.full(M * rld + off, 4, kind)
            r[off:].reshape(M, rld)[:, :N] = rb
            rbuf = dev(ud, r)
            rd = At(rbuf, off * kind.itemsize)
    obuf = dev(ud, host)
    od = At(obuf, off * kind.itemsize)
    ud.i8_linear(cd, sd, wd, wsd, od, M, N, K, bias=bd, residual=od if in_place else rd, dtype=dtype, codes_ld=K + pad[0],
                 w_ld=K + pad[1], res_ld=rld, out_ld=old)
    ud.synchronize()
    got = obuf.download(host.shape, kind)
    assert np.all(got[:off] == 5) and np.all(got[off + M * old:] == 5)
    got = got[off:off + M * old].reshape(M, old)
    assert np.all(got[:, N:] == 5)
    return ref.from_bits(got[:, :N], dtype)


def check(ud, rng, M, N, K, dtype, bias=False, residual=False, full=False, **kw):
    draw = (lambda *s: rng.integers(-128, 128, s).astype(np.int8)) if full else \
        (lambda *s: np.clip(np.rint(40 * rng.standard_normal(s)), -127, 127).astype(np.int8))
    codes, w = draw(M, K), draw(N, K)
    scales = (rng.uniform(0.5, 2, M) * 0.02).astype(np.float32)
    w_scales = (rng.uniform(0.5, 2, N) * 0.002).astype(np.float32)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    r = ref.stored(4 * rng.standard_normal((M, N)), dtype)[1] if residual else None
    got = run(ud, codes, scales, w, w_scales, dtype, b, r, in_place=residual and kw.pop("in_place", False), **kw)
    want, mag = ref.product(codes, scales, w, w_scales, b, r)
    # the sum to fp32, two scales, bias, residual: five roundings of what is at most mag; then the output's
    tol = 5 * ref.STEP32 * 1.01 * mag + ref.HALF_STEP[dtype] * 1.01 * np.abs(want) + ref.FLOOR[dtype]
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()


ROWS = [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 100, 128, 129, 200, 256, 300, 513]


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows(gpu, dtype, M):
    rng = np.random.default_rng([M, len(dtype)])
    check(gpu, rng, M, 256, 512, dtype)
    check(gpu, rng, M, 131, 272, dtype, bias=True, residual=True, off=1)
    check(gpu, rng, M, 515, 1040, dtype, residual=True, in_place=True, pad=(16, 32, 0, 3))
    check(gpu, rng, M, 1, 16, dtype, bias=True)


@pytest.mark.parametrize("K", [16, 48, 64, 80, 112, 128, 144, 240, 256, 272, 496, 512, 528, 1024, 4096, 4112, 12288])
@pytest.mark.parametrize("M", [1, 40, 150, 400])
def test_depths(gpu, M, K):
    rng = np.random.default_rng([M, K])
    check(gpu, rng, M, 200, K, "f32", full=True)
    check(gpu, rng, M, 77, K, "bf16", bias=True, pad=(16, 0, 0, 1))


@pytest.mark.parametrize("K", [16, 112, 128, 144, 496, 512, 528, 1008, 1024, 1040, 1152, 2064])
@pytest.mark.parametrize("M,N", [(16, 500), (30, 3001), (60, 4001), (125, 4001)])
def test_depths_shared_by_waves(gpu, M, N, K):
    """Blocks of 128 of k that do not come out even over the waves, or fewer than these; ends within a block."""
    check(gpu, np.random.default_rng([M, K]), M, N, K, "f32", bias=True, full=True, pad=(16, 0, 0, 0))


@pytest.mark.parametrize("N", [3, 15, 17, 31, 33, 64, 127, 129, 255, 257, 1025, 6144])
@pytest.mark.parametrize("M", [1, 20, 64, 140, 270])
def test_channels(gpu, M, N):
    rng = np.random.default_rng([M, N])
    check(gpu, rng, M, N, 320, "bf16", bias=True)
    check(gpu, rng, M, N, 256, "f16", residual=True, pad=(0, 16, 1, 2))


# every kernel of csrc/linear_plan.hpp, over grids of several tiles, none whole at the edges
TILES = [(3, 5001, 2064), (16, 1000, 8208), (2, 20003, 528), (30, 3001, 1040), (64, 4099, 656), (60, 9003, 272), (120, 6002, 400), (500, 6007, 784),
         (1000, 9001, 272), (2049, 5500, 144), (2500, 4001, 400), (4050, 4030, 272), (8200, 1500, 256), (130, 30001, 64), (700, 9000, 400),
         (60, 17003, 272), (130, 8003, 400), (300, 9001, 16), (2060, 5400, 48), (520, 3001, 112), (4, 700, 8208), (3, 9001, 2064), (16, 9001, 400),
         (63, 4001, 656), (29, 9001, 2064), (33, 4090, 16), (127, 4001, 2064), (9, 4095, 144), (17, 2003, 12304), (445, 4140, 960)]


@pytest.mark.parametrize("M,N,K", TILES)
def test_many_tiles(gpu, M, N, K):
    rng = np.random.default_rng([M, N])
    check(gpu, rng, M, N, K, "bf16", bias=True)
    check(gpu, rng, M, N, K, "f32", residual=True, full=True, pad=(0, 16, 3, 1))
    check(gpu, rng, M, N, K, "f16", bias=True, residual=True, in_place=True, off=3, pad=(32, 0, 0, 0))


@pytest.mark.parametrize("M", [1, 64, 200, 2100])
def test_largest_sums(gpu, M):
    """All codes -128: 128 * 128 * 131056 is the largest sum, 2^31 less 2^18."""
    K, N = 131056, 40 if M < 2000 else 6000
    codes, w = np.full((M, K), -128, np.int8), np.full((N, K), -128, np.int8)
    w[1::2] = 127
    got = run(gpu, codes, np.ones(M), w, np.ones(N), "f32")
    want = np.where(np.arange(N) % 2, -128 * 127 * K, 128 * 128 * K).astype(np.float64)
    assert np.all(np.abs(got - want) <= ref.STEP32 * np.abs(want))


@pytest.mark.parametrize("M", [1, 64, 260])
def test_scales_that_are_no_numbers(gpu, M):
    """A row whose scale is NaN is NaN and touches no other; a channel's likewise."""
    rng = np.random.default_rng(M)
    codes = rng.integers(-127, 128, (M, 128)).astype(np.int8)
    w = rng.integers(-127, 128, (70, 128)).astype(np.int8)
    scales, w_scales = np.ones(M), np.ones(70)
    scales[M // 2], w_scales[69] = np.nan, np.nan
    got = run(gpu, codes, scales, w, w_scales, "bf16")
    nan = np.zeros((M, 70), bool)
    nan[M // 2], nan[:, 69] = True, True
    np.testing.assert_array_equal(np.isnan(got), nan)
    want = codes.astype(np.float64) @ w.astype(np.float64).T
    assert np.all((np.abs(got - want) <= 2.0 ** -8 * 1.01 * np.abs(want))[~nan])


def test_half_saturates(gpu):
    codes, w = np.full((3, 64), 127, np.int8), np.full((20, 64), 127, np.int8)
    got = run(gpu, codes, np.array([1.0, -1.0, 1e-3]), w, np.ones(20), "f16")
    assert np.all(got[0] == 65504) and np.all(got[1] == -65504) and np.all(np.abs(got[2] - 1032.256) <= 0.51)


def test_no_rows(gpu):
    b = dev(gpu, np.zeros(64, np.float32))
    gpu.i8_linear(b, b, b, b, b, 0, 4, 16)
