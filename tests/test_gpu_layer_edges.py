"""The calls of include/ud_layer.h at their far ends: rows so far apart that their offsets pass 32 bits, the largest lds, histories
without penalties, every dtype's in-place forms over one row."""
import numpy as np
import pytest

import layer_ref as ref
from test_gpu_rows import NORM_REL

pytestmark = pytest.mark.gpu


class Rows:
    """Rows of `dtype` storage `ld` elements apart in a buffer of their own."""

    def __init__(self, ud, rows, width, ld, dtype):
        self.ud, self.shape, self.ld, self.dtype = ud, (rows, width), ld, np.dtype(dtype)
        self.buf = ud.DeviceBuffer(((rows - 1) * ld + width) * self.dtype.itemsize)
        self.ptr, self.nbytes = self.buf.ptr, self.buf.nbytes

    def put(self, a):
        a = np.ascontiguousarray(a, self.dtype)
        for i, r in enumerate(a):
            self.ud._check(self.ud.lib().ud_memcpy_htod(self.ptr + i * self.ld * self.dtype.itemsize, r.ctypes.data, r.nbytes))
        return self

    def get(self):
        out = np.empty(self.shape, self.dtype)
        for i in range(len(out)):
            self.ud._check(self.ud.lib().ud_memcpy_dtoh(out[i].ctypes.data, self.ptr + i * self.ld * self.dtype.itemsize, out[i].nbytes))
        return out


def dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


@pytest.mark.parametrize("eight", [False, True])
def test_norm_rows_far_apart(gpu, eight):
    """Ten rows 2^28 elements apart: the last lies 4.5 GiB behind the first (codes 2.3 GiB)."""
    ud, rng, rows, dim, ld = gpu, np.random.default_rng(1), 10, 520, 1 << 28
    bits, x = ref.stored(rng.standard_normal((rows, dim)), "bf16")
    xd = Rows(ud, rows, dim, ld, np.uint16).put(bits)
    od = Rows(ud, rows, dim, ld, np.int8) if eight else xd
    sd = dev(ud, np.zeros(rows, np.float32)) if eight else None
    ud.rms_norm(xd, od, rows, dim, scales=sd, out_dtype="i8" if eight else None, x_ld=ld, out_ld=ld)
    ud.synchronize()
    y = ref.normed(x, None, float(np.float32(1e-6)))
    if eight:
        ref.check_codes(od.get(), sd.download(rows).astype(np.float64), y, NORM_REL)
    else:
        got = ref.from_bits(od.get(), "bf16")
        assert np.all(np.abs(got - y) <= (2.0 ** -8 * 1.01 + NORM_REL) * np.abs(y))


@pytest.mark.parametrize("M,N,K", [(3, 1100, 64), (1100, 130, 80), (1030, 1100, 144), (40, 1100, 400), (24, 2100, 272)])
def test_products_of_rows_far_apart(gpu, M, N, K):
    """Rows 2^22 bytes apart, the largest distance: over a thousand of them pass 4 GiB."""
    ud, rng, ld = gpu, np.random.default_rng([M, N]), 1 << 22
    c, w = rng.integers(-127, 128, (M, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    cd, wd = Rows(ud, M, K, ld if M > 1000 else K, np.int8).put(c), Rows(ud, N, K, ld if N > 1000 else K, np.int8).put(w)
    s, ws = rng.uniform(0.5, 2, M).astype(np.float32), rng.uniform(0.5, 2, N).astype(np.float32)
    out = ud.DeviceBuffer(4 * M * N)
    ud.i8_linear(cd, dev(ud, s), wd, dev(ud, ws), out, M, N, K, dtype="f32", codes_ld=cd.ld, w_ld=wd.ld)
    ud.synchronize()
    want, mag = ref.product(c, s, w, ws)
    assert np.all(np.abs(out.download((M, N)) - want) <= 4 * ref.STEP32 * mag)


@pytest.mark.parametrize("M", [9, 400])
def test_product_into_rows_far_apart(gpu, M):
    ud, rng, N, K = gpu, np.random.default_rng(M), 700, 96
    ld = 1 << 28 if M < 100 else 6_000_001
    c, w = rng.integers(-127, 128, (M, K)).astype(np.int8), rng.integers(-127, 128, (N, K)).astype(np.int8)
    bits, r = ref.stored(100 * rng.standard_normal((M, N)), "bf16")
    od = Rows(ud, M, N, ld, np.uint16).put(bits)
    s, ws = rng.uniform(0.5, 2, M).astype(np.float32) * 1e-2, rng.uniform(0.5, 2, N).astype(np.float32) * 1e-1
    ud.i8_linear(dev(ud, c), dev(ud, s), dev(ud, w), dev(ud, ws), od, M, N, K, residual=od, res_ld=ld, out_ld=ld)
    ud.synchronize()
    want, mag = ref.product(c, s, w, ws, None, r)
    got = ref.from_bits(od.get(), "bf16")
    assert np.all(np.abs(got - want) <= 5 * ref.STEP32 * mag + 2.0 ** -8 * 1.01 * np.abs(want))


@pytest.mark.parametrize("n,V", [(20, 3000), (20, 40000)])
def test_logits_far_apart(gpu, n, V):
    """Rows 2^27 elements apart: 5 GiB of bf16, 10 of fp32, the mask's 2^26 words."""
    ud, rng, ld = gpu, np.random.default_rng(V), 1 << 27
    bits, x = ref.stored(rng.standard_normal((n, V)), "bf16")
    allowed = rng.random((n, V)) < 0.5
    words = -(-V // 32)
    ind, od = Rows(ud, n, V, ld, np.uint16).put(bits), Rows(ud, n, V, ld, np.float32)
    md = Rows(ud, n, words, 1 << 26, np.uint32).put(ref.mask_words(allowed))
    token, ws = ud.DeviceBuffer(4 * n), ud.DeviceBuffer(ud.logits_workspace_bytes(n, V))
    ud.logits_process(ind, od, n, V, token=token, mask=md, n_masks=n, workspace=ws, dtype="bf16", ld=ld, out_ld=ld, mask_ld=1 << 26)
    ud.synchronize()
    want = np.where(allowed, x, -np.inf)
    np.testing.assert_array_equal(od.get(), want)
    np.testing.assert_array_equal(token.download(n, np.int32), ref.chosen(want))


def test_histories_without_penalties(gpu):
    """Penalties are 1, 0, 0 where they are not given; logits in place; no token asked for, no workspace."""
    ud, rng = gpu, np.random.default_rng(3)
    x = rng.standard_normal((2, 500)).astype(np.float32)
    xd = dev(ud, x)
    ud.logits_process(xd, xd, 2, 500, tokens=dev(ud, np.arange(50, dtype=np.int32)), n_tokens=50, ranges=dev(ud, np.array([[0, 5, 50]] * 2, np.int32)))
    ud.synchronize()
    np.testing.assert_array_equal(xd.download((2, 500)), x)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_one_row_in_place(gpu, dtype):
    """One row may be normed in place whatever its lds are, the sums into the residual."""
    ud, rng, dim = gpu, np.random.default_rng(4), 264
    (xb, x), (rb, r) = (ref.stored(rng.standard_normal((1, dim)), dtype) for _ in range(2))
    xd, rd = dev(ud, xb), dev(ud, rb)
    ud.rms_norm(xd, xd, 1, dim, residual=rd, sum_out=rd, dtype=dtype, x_ld=dim, out_ld=dim + 64, sum_ld=dim + 8)
    ud.synchronize()
    s = ref.summed(x, r, dtype)
    np.testing.assert_array_equal(ref.from_bits(rd.download((1, dim), xb.dtype), dtype), s)
    y = ref.normed(s, None, float(np.float32(1e-6)))
    got = ref.from_bits(xd.download((1, dim), xb.dtype), dtype)
    assert np.all(np.abs(got - y) <= (ref.HALF_STEP[dtype] * 1.01 + NORM_REL) * np.abs(y) + ref.FLOOR[dtype])
