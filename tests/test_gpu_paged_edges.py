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
