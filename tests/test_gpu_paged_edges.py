"""GPU tests of the paged-cache operators at the edges of what their header allows (include/ud_decode.h)."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def _dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


class At:
    def __init__(self, buf, off):
        self.buf, self.ptr = buf, buf.ptr + off


@pytest.mark.parametrize("rows", [1, 5])
@pytest.mark.parametrize("place", ["behind", "between", "before", "in place"])
def test_append_outputs_beside_inputs(gpu, rows, place):
    """q_out in the gaps of the fused rows [gap | q | gap | k | v], rows of one distance: its rows come out right and k, v and the
    other gap are as they were."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(91), 4, 2, 64
    qw, kw = hq * d, hkv * d
    ld = 3 * qw + 2 * kw
    q0, k0 = qw, 3 * qw
    v0 = k0 + kw
    out0 = {"behind": 0, "between": 2 * qw, "before": 0, "in place": q0}[place]
    x = ref.rounded(rng.standard_normal((rows, ld)), "bf16")
    src = _dev(ud, ref.to_bits(x, "bf16"))
    out = At(src, out0 * 2)
    if place == "behind":                                # as "between", the whole a row on: the last row behind the last input
        src = _dev(ud, ref.to_bits(np.concatenate([x, x[:1]]), "bf16"))
        out = At(src, (ld) * 2)                      # the first gap of the next row
        out0 = 0
    table, num = ref.assign_pages(rng, [rows])
    kp, vp = (_dev(ud, ref.new_pool("bf16", num, hkv, d)) for _ in range(2))
    pos, seqs, inv = np.arange(rows, dtype=np.int32), np.zeros(rows, np.int32), ud.rope_inv_freq(d)
    bt, pd, sd, iv = _dev(ud, table), _dev(ud, pos), _dev(ud, seqs), _dev(ud, inv)
    ud.qk_norm_rope_append(At(src, q0 * 2), At(src, k0 * 2), At(src, v0 * 2), out, kp, vp, num, bt, 1, table.shape[1], pd, rows, hq, hkv, d,
                           seqs=sd, inv_freq=iv, q_ld=ld, k_ld=ld, v_ld=ld, q_out_ld=ld)
    kb, vb = ud.DeviceBuffer(rows * kw * 2), ud.DeviceBuffer(rows * kw * 2)
    ud.paged_kv_read(kp, vp, num, bt, 1, table.shape[1], pd, kb, vb, rows, hkv, d, seqs=sd, dtype="bf16")
    ud.synchronize()
    after = ref.from_bits(src.download((rows + (place == "behind"), ld), np.uint16), "bf16")
    first = 1 if place == "behind" else 0
    got = after[first:first + rows, out0:out0 + qw].reshape(rows, hq, d)
    want = ref.norm_rope(x[:, q0:q0 + qw].reshape(rows, hq, d), None, 0, pos, inv)
    # sine and cosine rounded to fp32, two products and a sum: 5 roundings of the pair's length; then to bf16
    amp = np.sqrt(2) * np.abs(x[:, q0:q0 + qw]).max()
    assert np.all(np.abs(got - want) <= ref.HALF_STEP["bf16"] * np.abs(want) * 1.01 + 5 * 2.0 ** -24 * amp)
    expect = np.concatenate([x, x[:1]]) if place == "behind" else x.copy()
    expect[first:first + rows, out0:out0 + qw] = got.reshape(rows, -1)
    np.testing.assert_array_equal(after, expect)
    np.testing.assert_array_equal(ref.from_bits(vb.download((rows, kw), np.uint16), "bf16"), x[:, v0:])
    want_k = ref.norm_rope(x[:, k0:v0].reshape(rows, hkv, d), None, 0, pos, inv).reshape(rows, -1)
    got_k = ref.from_bits(kb.download((rows, kw), np.uint16), "bf16")
    assert np.all(np.abs(got_k - want_k) <= ref.HALF_STEP["bf16"] * np.abs(want_k) * 1.01 + 5 * 2.0 ** -24 * np.sqrt(2) * np.abs(x).max())


@pytest.mark.parametrize("norm", [False, True])
def test_fp4_keys_past_fp32_saturate(gpu, norm):
    """Finite rows whose normalised and rotated keys pass fp32's range: the largest code and exponent, not a block of NaN; the
    other blocks, and blocks of infinities and NaN, as ever."""
    ud, rng, d = gpu, np.random.default_rng(92), 128
    rows, big = 6, float(np.float32(3.3e38))
    x = rng.standard_normal((rows, 2, d))
    weight = None
    pos, inv = np.arange(rows) * 7 + 1, ud.rope_inv_freq(d)
    if norm:
        weight = np.ones(d, np.float32)
        weight[[3, 40, 67, 100]] = 3e38                  # times up to sqrt(d): past fp32
        x[:, 0, 3], x[:, 0, 100] = 9, -7
    else:
        x[:, 0, 0], x[:, 0, 64] = big, -big              # rotated by pos: up to 1.41 times as long
        x[1, 0, 70], x[1, 0, 6] = big, big
        x[2, 0, 33], x[3, 0, 97] = np.inf, np.nan
    x = ref.rounded(x, "f32")
    table, num = ref.assign_pages(rng, [int(p) + 1 for p in pos])
    kp, vp = (_dev(ud, ref.new_pool("mxfp4", num, 1, d)) for _ in range(2))
    k, v, bt, pd, iv = (_dev(ud, a) for a in (x[:, 0].astype(np.float32), x[:, 1].astype(np.float32), table, pos.astype(np.int32), inv))
    ud.qk_norm_rope_append(None, k, v, None, kp, vp, num, bt, rows, table.shape[1], pd, rows, 0, 1, d, inv_freq=iv, dtype="f32",
                           kv_format="mxfp4", k_weight=None if weight is None else _dev(ud, weight))
    kb, vb = ud.DeviceBuffer(rows * d * 4), ud.DeviceBuffer(rows * d * 4)
    ud.paged_kv_read(kp, vp, num, bt, rows, table.shape[1], pd, kb, vb, rows, 1, d, kv_format="mxfp4")
    ud.synchronize()
    with np.errstate(invalid="ignore"):
        want = ref.norm_rope(x[:, :1], weight, 1e-6, pos, inv)
    finite = np.isfinite(want)
    assert np.abs(want[finite]).max() > 3.41e38
    np.testing.assert_array_equal(kb.download((rows, 1, d)), ref.held(want, "mxfp4"))
    np.testing.assert_array_equal(vb.download((rows, 1, d)), ref.held(x[:, 1:], "mxfp4"))
