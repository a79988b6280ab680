"""GPU parity of ud_qk_norm_rope_append and ud_paged_kv_read with their float64 forms (paged_ref.py): every row type and
page format, both head sizes, groups of 1 to 8, strided rows, far positions, MXFP4's ties and borders, padding rows."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu


def _dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def run(ud, x, lens, dtype, fmt, hq, hkv, d, pos, seqs, weights=(None, None), inv=None, eps=1e-6, fused=True, in_place=False, table=None,
        num=None, rng=None):
    """x [rows, hq + 2 hkv, d] float64 (values of dtype).  Returns q out, the pool's K and V after the call, what they were
    before, and what paged_kv_read gives."""
    rows = len(x)
    if table is None:
        table, num = ref.assign_pages(rng, lens)
    n, most = table.shape
    raw = ref.to_bits(x, dtype).reshape(rows, -1)
    before_k, before_v = (rng.integers(0, 255, ref.new_pool(fmt, num, hkv, d).shape).astype(np.uint8) for _ in range(2))
    kp, vp = _dev(ud, before_k), _dev(ud, before_v)
    size = raw.dtype.itemsize
    pad = 0 if fused else 8

    class At:
        def __init__(self, buf, off):
            self.buf, self.ptr = buf, buf.ptr + off

    if fused:
        src = _dev(ud, raw)
        ld = raw.shape[1]
        q, k, v = At(src, 0), At(src, hq * d * size), At(src, (hq + hkv) * d * size)
        lds = dict(q_ld=ld, k_ld=ld, v_ld=ld)
    else:
        cut = [raw[:, :hq * d], raw[:, hq * d:(hq + hkv) * d], raw[:, (hq + hkv) * d:]]
        q, k, v = (_dev(ud, np.concatenate([c, np.zeros((rows, pad), c.dtype)], 1)) for c in cut)
        lds = dict(q_ld=hq * d + pad, k_ld=hkv * d + pad, v_ld=hkv * d + pad)
    if in_place:
        out, old = q, lds["q_ld"]
    else:
        old = hq * d + 4
        out = _dev(ud, np.full((rows, old), 7, raw.dtype))
    opt = lambda a: None if a is None else _dev(ud, a)  # noqa: E731
    posd, seqd, bt = _dev(ud, pos.astype(np.int32)), opt(None if seqs is None else seqs.astype(np.int32)), _dev(ud, table)
    qw, kw, iv = opt(weights[0]), opt(weights[1]), opt(inv)
    ud.qk_norm_rope_append(q, k, v, out, kp, vp, num, bt, n, most, posd, rows, hq, hkv, d, seqs=seqd, q_weight=qw, k_weight=kw, eps=eps,
                           inv_freq=iv, dtype=dtype, kv_format=fmt, q_out_ld=old, **lds)
    back = "f32" if fmt == "mxfp4" else fmt
    kb, vb = (_dev(ud, np.full((rows, hkv * d), 9, np.float32)) for _ in range(2))
    ud.paged_kv_read(kp, vp, num, bt, n, most, posd, kb, vb, rows, hkv, d, seqs=seqd, dtype=back, kv_format=fmt)
    ud.synchronize()
    store = np.float32 if back == "f32" else np.uint16
    read = [ref.from_bits(b.download((rows, hkv, d), store), back) for b in (kb, vb)]
    width = old if not in_place or not fused else raw.shape[1]
    got = (out.buf if in_place and fused else out).download((rows, width), raw.dtype)[:, :hq * d].reshape(rows, hq, d)
    pools = [b.download(before_k.shape, np.uint8) for b in (kp, vp)]
    return ref.from_bits(got, dtype), pools, (before_k, before_v), read, table, num


def check(ud, rng, dtype, fmt, hq, hkv, d, rows_per, past, norm, rope, fused=True, in_place=False):
    lens = [p + t for p, t in zip(past, rows_per)]
    pos = np.concatenate([p + np.arange(t) for p, t in zip(past, rows_per)])
    seqs = np.repeat(np.arange(len(lens)), rows_per)
    order = rng.permutation(len(pos))
    pos, seqs = pos[order], seqs[order]
    x = ref.rounded(rng.standard_normal((len(pos), hq + 2 * hkv, d)) * np.exp(rng.standard_normal((1, 1, d))), dtype)
    w = [(1 + 0.3 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    inv = ud.rope_inv_freq(d) if rope else None
    q, pools, before, read, table, num = run(ud, x, lens, dtype, fmt, hq, hkv, d, pos, seqs, w, inv, fused=fused, in_place=in_place, rng=rng)
    want_q = ref.norm_rope(x[:, :hq], w[0], 1e-6, pos, inv)
    want_k = ref.norm_rope(x[:, hq:hq + hkv], w[1], 1e-6, pos, inv)
    # fp32: the sum of d squares (each lane adds 8, then a tree of 4), a root, a division, three products and a sum:
    # under 16 roundings of a value no larger than the pair that is rotated
    def amp(y):
        a = np.hypot(y[..., :d // 2], y[..., d // 2:])
        return np.concatenate([a, a], -1)
    tol = lambda y, t: ref.HALF_STEP[t] * np.abs(y) * 1.01 + 16 * 2.0 ** -24 * amp(y) + 2.0 ** -25  # noqa: E731
    assert np.all(np.abs(q - want_q) <= tol(want_q, dtype))
    want_v = ref.held(x[:, hq + hkv:], fmt)
    np.testing.assert_array_equal(read[1], want_v)
    if fmt == "mxfp4":
        np.testing.assert_array_equal(read[0], ref.held(want_k, fmt))
    else:
        assert np.all(np.abs(read[0] - want_k) <= tol(want_k, fmt))
    # the pages hold what was read, at the documented places, and nothing else of them has changed
    expect = [b.copy() for b in before]
    for t in range(len(pos)):
        page, row = table[seqs[t], pos[t] // 16], pos[t] % 16
        for e, r, p in zip(expect, read, pools):
            np.testing.assert_array_equal(ref.get_row(p, fmt, d, page, row), r[t])
            ref.put_row(e, fmt, d, page, row, r[t])
            if fmt == "mxfp4":                       # a zero's sign, and a block without its largest value, are not in the values
                a = slice(row * d // 2, (row + 1) * d // 2)
                e[page, :, a] = p[page, :, a]
                a = slice(8 * d + row * d // 32, 8 * d + (row + 1) * d // 32)
                e[page, :, a] = p[page, :, a]
    for e, p in zip(expect, pools):
        np.testing.assert_array_equal(e, p)


@pytest.mark.parametrize("dtype,fmt", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f16"), ("bf16", "mxfp4"),
                                       ("f16", "mxfp4"), ("f32", "mxfp4")])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (7, 1, 128), (16, 2, 64), (5, 5, 64)])
def test_types_and_heads(gpu, dtype, fmt, hq, hkv, d):
    rng = np.random.default_rng([hq, d, len(dtype), len(fmt)])
    check(gpu, rng, dtype, fmt, hq, hkv, d, [1, 17, 3], [0, 15, 130], True, True)
    check(gpu, rng, dtype, fmt, hq, hkv, d, [2, 5], [31, 0], False, True, fused=False, in_place=True)
    check(gpu, rng, dtype, fmt, hq, hkv, d, [1], [7], True, False, fused=False)
    check(gpu, rng, dtype, fmt, hq, hkv, d, [1, 1, 1], [47, 0, 16], False, False, in_place=True)


@pytest.mark.parametrize("dtype,fmt", [("f32", "f16"), ("bf16", "mxfp4")])
def test_far_positions(gpu, dtype, fmt):
    """A million tokens on, an fp32 angle would be off by 0.03 rad."""
    check(gpu, np.random.default_rng(5), dtype, fmt, 4, 2, 128, [3, 2], [999_983, 131_071], True, True)


def test_sequences_by_row_and_no_queries(gpu):
    """seqs = None: row t is sequence t; q_heads = 0 appends keys and values alone."""
    ud, rng, hkv, d = gpu, np.random.default_rng(6), 2, 64
    pos = np.array([5, 0, 40])
    x = ref.rounded(rng.standard_normal((3, 2 * hkv, d)), "f16")
    q, pools, before, read, table, num = run(ud, x, [6, 1, 41], "f16", "mxfp4", 0, hkv, d, pos, None, rng=rng)
    np.testing.assert_array_equal(read[0], ref.held(x[:, :hkv], "mxfp4"))
    np.testing.assert_array_equal(read[1], ref.held(x[:, hkv:], "mxfp4"))


def test_padding_rows_leave_everything(gpu):
    """Rows of no sequence, of a position below 0 or past the table, or of a page that is not held: nothing is written, q
    included, and reading them gives 0."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(7), 4, 2, 128
    table, num = ref.assign_pages(rng, [40, 40], keep=lambda i, b: (i, b) != (1, 1))
    pos = np.array([3, -1, 48, 3, 3, 20, 2 ** 31 - 1, 21])
    seqs = np.array([0, 0, 0, 2, -1, 1, 0, 0])
    real = np.array([1, 0, 0, 0, 0, 0, 0, 1], bool)
    x = ref.rounded(rng.standard_normal((8, hq + 2 * hkv, d)), "bf16")
    for fmt in ("bf16", "mxfp4"):
        q, pools, before, read, _, _ = run(ud, x, None, "bf16", fmt, hq, hkv, d, pos, seqs, inv=ud.rope_inv_freq(d), table=table, num=num, rng=rng)
        untouched = ref.from_bits(np.full(1, 7, np.uint16), "bf16")[0]
        assert np.all(q[~real] == untouched) and np.all(q[real] != untouched)
        for r in read:
            assert np.all(r[~real] == 0) and np.any(r[real] != 0)
        for b, p in zip(before, pools):
            assert len({tuple(ix[:1]) for ix in np.argwhere(b != p)}) == 2      # two pages, a row each
            assert (b != p).reshape(num, hkv, -1).sum() <= 2 * hkv * (2 * d)


def test_fp4_borders(gpu):
    """Ties, the blocks' largest values at and around 7 x a power of two, zeros, tiny and huge values; a NaN or an infinity
    makes its block NaN and no other."""
    ud, rng, d = gpu, np.random.default_rng(8), 128
    mid = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 7, 6, 0, .5, 4, 7 * (1 - 2.0 ** -23), 5 * (1 + 2.0 ** -22), .25 * (1 - 2.0 ** -23), 3])
    x = np.zeros((6, 2, d))
    for h in range(2):
        x[0, h] = np.concatenate([mid, -mid] * 4)
        x[1, h] = x[0, h] * 2.0 ** -30
        x[2, h, 0::32] = [7 * (1 + 2.0 ** -23), 7 * 2.0 ** 60, 2.0 ** -99, 3e38]
        x[3, h] = rng.standard_normal(d) * np.repeat([1e-38, 1e-30, 1e30, 1], 32)
        x[5, h] = rng.standard_normal(d)
    x = ref.rounded(x, "f32")
    x[4, 0, 5], x[4, 0, 70], x[4, 1, 127] = np.nan, np.inf, -np.inf
    q, pools, before, read, table, num = run(ud, x, [1] * 6, "f32", "mxfp4", 0, 1, d, np.zeros(6, int), None, rng=rng)
    np.testing.assert_array_equal(read[0], ref.held(x[:, :1], "mxfp4"))
    np.testing.assert_array_equal(read[1], ref.held(x[:, 1:], "mxfp4"))
    assert np.isnan(read[0][4]).sum() == 64 and np.isnan(read[1][4]).sum() == 32


def test_read_as_bf16(gpu):
    """MXFP4's values are bf16 values; half and bf16 pages also read as fp32."""
    ud, rng, hkv, d = gpu, np.random.default_rng(9), 3, 64
    for fmt, back in [("mxfp4", "bf16"), ("f16", "f32"), ("bf16", "f32")]:
        table, num = ref.assign_pages(rng, [20])
        x = ref.held(rng.standard_normal((20, hkv, d)), fmt)
        pools = [ref.new_pool(fmt, num, hkv, d) for _ in range(2)]
        ref.fill(pools[0], table, fmt, d, [x], num)
        ref.fill(pools[1], table, fmt, d, [-x], num)
        out = [ud.DeviceBuffer(20 * hkv * d * 4) for _ in range(2)]
        ud.paged_kv_read(_dev(ud, pools[0]), _dev(ud, pools[1]), num, _dev(ud, table), 1, table.shape[1], _dev(ud, np.arange(20, dtype=np.int32)),
                         out[0], out[1], 20, hkv, d, seqs=_dev(ud, np.zeros(20, np.int32)), dtype=back, kv_format=fmt)
        ud.synchronize()
        for o, want in zip(out, (x, -x)):
            got = ref.from_bits(o.download((20, hkv, d), np.uint16 if back == "bf16" else np.float32), back)
            np.testing.assert_array_equal(got, want)
