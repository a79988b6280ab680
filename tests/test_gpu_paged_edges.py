"""GPU tests of the paged-cache operators at the edges of what their header allows (include/ud_decode.h)."""
import numpy as np
import pytest

import paged_ref as ref
from test_gpu_paged_window import P_STEP, PROMPT_STEP, PROMPTS, TYPES, Cache, causal, close, prefill, window

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


def _infinite_values(ud, fmt, keys, d, low):
    """A cache whose values are infinite in places: channel 1 +inf at key 5, 2 -inf at key 70, 3 both, 4 a NaN, 5 +inf at key 80, 6 +inf
    near the end.  The scores of key 80 and of the first `low` keys, of queries along e, are so far below the rest's that their
    probabilities, about exp(-300), are 0 in fp32."""
    rng, hkv = np.random.default_rng([93, keys, d]), 2
    e = rng.standard_normal(d)
    e /= np.linalg.norm(e)
    k, v = 0.3 * rng.standard_normal((keys, hkv, d)), rng.standard_normal((keys, hkv, d))
    far = -300 * np.sqrt(d) / 8
    k[:low] += far * e
    k[80] = far * e
    v[5, :, 1] = v[5, :, 3] = v[80, 0, 5] = v[keys - 25, 1, 6] = np.inf
    v[70, :, 2] = v[70, :, 3] = -np.inf
    v[70, 1, 4] = np.nan
    return e, Cache(ud, rng, fmt, [keys], hkv, d, k=[ref.held(k, fmt)], v=[ref.held(v, fmt)])


def _check_infinite(got, want, c, d, dtype, p_step):
    """Outputs are infinite or NaN exactly where the formula's are (p > 0: an infinity however small p is), half ones saturated;
    the others within their tolerance."""
    out, mag, top, dot, count = want
    got = got.reshape(out.shape).copy()
    odd = ~np.isfinite(out)
    assert np.isposinf(out).any() and np.isneginf(out).any() and np.isnan(out).any() and not odd[..., 7:].any()
    np.testing.assert_array_equal(got[odd], np.clip(out[odd], -65504, 65504) if dtype == "f16" else out[odd])
    got[odd] = 0
    close(got, (np.where(odd, 0, out), np.where(odd, 0, mag), top, dot, count), c, d, dtype, p_step)


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("d,group,keys,low", [(128, 1, 160, 0), (64, 7, 160, 0), (128, 4, 6000, 2000), (64, 2, 6000, 2000)])
def test_infinite_values_that_are_seen(gpu, fmt, dtype, d, group, keys, low):
    """An infinity among a row's values makes its output that infinity, whether the other rows of the workgroup see its page whole
    or in part."""
    ud, hq, M = gpu, 2 * group, 3
    e, c = _infinite_values(ud, fmt, keys, d, low)
    q = ref.rounded(np.random.default_rng(94).standard_normal((1, M, hq, d)) * 0.3 + 8 * e, dtype)
    for r in ([[0, keys]] * M, [[0, keys], [3, keys - 2], [37, keys - 31]], [[70, keys - 20], [71, keys], [9, 9]], [[0, keys], [0, 5], [5, 6]]):
        ranges = np.array([r])
        want = ref.attention(q[0], c.k, c.v, np.zeros(M, int), ranges[0], 4, 2, c.most * 16)
        got = window(ud, c, q, ranges, 4, dtype, span=keys)
        if r[0][0] == 70:                                # key 5 is not seen, nor key 70 by the second row
            assert not np.isposinf(want[0][..., :4]).any()
        _check_infinite(got, want, c, d, dtype, P_STEP[fmt, dtype])


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("fmt", ["bf16", "f16"])
@pytest.mark.parametrize("d,keys,low,win", [(128, 160, 0, 0), (64, 320, 0, 260), (128, 6000, 2000, 0), (64, 6000, 2000, 5950)])
def test_infinite_values_that_prompts_see(gpu, fmt, d, keys, low, win):
    ud, hq, rows = gpu, 4, 70
    e, c = _infinite_values(ud, fmt, keys, d, low)
    q = ref.rounded(np.random.default_rng(95).standard_normal((rows, hq, d)) * 0.3 + 8 * e, fmt)
    whole = np.tile([0, keys // 16 * 16], (rows, 1))
    for ranges in (whole, causal([rows], [keys - rows], win)):
        want = ref.attention(q, c.k, c.v, np.zeros(rows, int), ranges, 2, 2, c.most * 16)
        got = prefill(ud, c, q, [0, rows], ranges, 2, fmt, span=keys)
        _check_infinite(got, want, c, d, fmt, PROMPT_STEP[fmt])


def test_half_queries_over_small_fp4_values(gpu):
    """Blocks below half's normal range: the prompt's values are the nearest multiples of 2^-24, the windowed call's the cached
    ones."""
    ud, d = gpu, 128
    v = np.zeros((1, 1, d))
    for b, e in enumerate((-22, -23, -24, -25)):
        v[0, 0, 32 * b:32 * b + 14] = np.concatenate([ref.LEVELS[1:], -ref.LEVELS[1:]]) * 2.0 ** e
    c = Cache(ud, np.random.default_rng(96), "mxfp4", [1], 1, d, k=[np.zeros((1, 1, d))], v=[v])
    got = prefill(ud, c, np.ones((1, 1, d)), [0, 1], np.array([[0, 1]]), 0, "f16")[0, 0]
    np.testing.assert_array_equal(got, v[0, 0].astype(np.float16).astype(np.float64))
    np.testing.assert_array_equal(got[:64], v[0, 0, :64])    # exponents -22 and -23 stay as they are
    assert (got[64:] != v[0, 0, 64:]).any()
    got = window(ud, c, np.ones((1, 1, 1, d)), np.array([[[0, 1]]]), 0, "f32")[0, 0, 0]
    np.testing.assert_array_equal(got, v[0, 0])


def test_half_queries_over_small_fp4_keys(gpu):
    """Keys of 2^-25 under queries near half's end: the prompt's scores are those of the keys rounded to half (all 0), the
    windowed call's those of the cached keys."""
    ud, rng, d, keys = gpu, np.random.default_rng(97), 64, 32
    sign = rng.choice([-1.0, 1.0], (keys, 1, 1))
    k = np.tile(sign * 2.0 ** -25, (1, 1, d))
    v = sign * rng.choice([1.0, 1.5, 2.0], (keys, 1, d))
    c = Cache(ud, rng, "mxfp4", [keys], 1, d, k=[k], v=[v])
    assert np.array_equal(ref.held(k, "mxfp4"), k) and np.array_equal(ref.held(v, "mxfp4"), v)
    q = ref.rounded(rng.uniform(30_000, 60_000, (2, 4, d)), "f16")
    ranges, seq = np.array([[0, keys], [3, keys]]), np.zeros(2, int)
    exact = ref.attention(q, c.k, c.v, seq, ranges, 0, 1, keys)
    half = ref.attention(q, [k.astype(np.float16).astype(np.float64)], c.v, seq, ranges, 0, 1, keys)
    assert np.abs(exact[0] - half[0]).min() > 2 * ref.attention_tolerance(*exact, d, "f16", PROMPT_STEP["f16"]).max()
    got = window(ud, c, q[None], ranges[None], 0, "f16")
    close(got, exact, c, d, "f16", P_STEP["mxfp4", "f16"])
    got = prefill(ud, c, q, [0, 2], ranges, 0, "f16")
    close(got, half, c, d, "f16", PROMPT_STEP["f16"])


def _huge(ud, fmt, dtype, d, q_log, k_log):
    """Keys and queries along one direction: scores of about 2^(q_log + k_log + 10.6) in binary digits that rise, fall and repeat
    over the keys, and whose largest is ahead of the next by 1 in 128 or more (or by nothing: equal keys)."""
    rng, keys, hkv, rows, hq = np.random.default_rng([98, q_log, abs(k_log), d]), 330, 2, 6, 4
    e = rng.choice([-1.0, 1.0], d)
    a = 64 + np.concatenate([np.arange(60), 40 - np.arange(40), rng.integers(0, 63, keys - 100)])
    a[[100, 217, 320]] = 127
    a[[150, 151]] = 63
    k = ref.held((a * 2.0 ** k_log)[:, None, None] * e * np.ones((1, hkv, 1)), fmt)
    c = Cache(ud, rng, fmt, [keys], hkv, d, k=[k])
    sign = rng.choice([-1.0, 1.0], (rows, hq, 1)) * np.array([1, 1.5, 1.25, 1.0, 1.75, 1.0])[:, None, None]
    return c, ref.rounded(sign * 2.0 ** q_log * e, dtype)


def _check_huge(got, want, dtype, p_step):
    """The mean of the values of the equal keys whose score is the largest: every other's probability is 0."""
    out, mag, top, dot, count = want
    assert np.all(np.abs(got.reshape(out.shape) - out) <= (p_step + 2.0 ** -20) * mag + ref.HALF_STEP[dtype] * np.abs(out) * 1.01 + 2.0 ** -25)


HUGE = {"f16": [(5, 0), (10, 1), (12, 4), (14, 8)], "bf16": [(5, 0), (9, 0), (12, 4), (20, 10), (40, 30), (55, 50)]}


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_huge_scores(gpu, fmt, dtype, d):
    """Scores up to 2^115, where one step of fp32 is far more than the exponents that a probability has room for."""
    ud = gpu
    for q_log, k_log in HUGE["f16" if "f16" in (fmt, dtype) else "bf16"]:
        c, q = _huge(ud, fmt, dtype, d, q_log, k_log)
        ranges = np.array([[0, 330], [0, 330], [3, 217], [150, 320], [50, 160], [99, 152]])
        want = ref.attention(q, c.k, c.v, np.zeros(6, int), ranges, 0, 2, c.most * 16)
        _check_huge(window(ud, c, q[None], ranges[None], 0, dtype), want, dtype, P_STEP[fmt, dtype])
        split = window(ud, c, q[None], ranges[None], 0, dtype, span=100_000)      # (many splits, most of them empty)
        _check_huge(split, want, dtype, P_STEP[fmt, dtype])


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
@pytest.mark.parametrize("d", [64, 128])
def test_huge_scores_of_prompts(gpu, fmt, dtype, d):
    ud = gpu
    for q_log, k_log in HUGE["f16" if "f16" in (fmt, dtype) else "bf16"]:
        c, q = _huge(ud, fmt, dtype, d, q_log, k_log)
        q = np.tile(q, (50, 1, 1))
        ranges = causal([300], [30], 0)
        want = ref.attention(q, c.k, c.v, np.zeros(300, int), ranges, 0, 2, c.most * 16)
        for span in (330, 20_000):
            _check_huge(prefill(ud, c, q, [0, 300], ranges, 0, dtype, span=span), want, dtype, PROMPT_STEP[dtype])


@pytest.mark.parametrize("fmt,dtype", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("mxfp4", "bf16")])
def test_huge_scores_in_all_directions(gpu, fmt, dtype):
    """Random keys and queries up to half's end: outputs are mixtures of the values that a row sees, none infinite or NaN, none 0 for
    want of a probability."""
    ud, rng, d, keys = gpu, np.random.default_rng(99), 64, 700
    for size in (600, 2_500, 9_000):
        k = [ref.held(np.clip(rng.standard_normal((keys, 1, d)) * size, -60_000, 60_000), fmt)]
        v = [ref.held(1 + rng.random((keys, 1, d)), fmt)]
        c = Cache(ud, rng, fmt, [keys], 1, d, k=k, v=v)
        q = ref.rounded(np.clip(rng.standard_normal((70, 8, d)) * size, -60_000, 60_000), dtype)
        ends = keys - 69 + np.arange(70)
        ranges = np.stack([0 * ends, ends], -1)
        got = [window(ud, c, q[None, 62:], ranges[None, 62:], 0, dtype), window(ud, c, q[None, :5], ranges[None, :5], 0, dtype, span=50_000)]
        if dtype != "f32":
            got += [prefill(ud, c, q, [0, 70], ranges, 0, dtype, span=s) for s in (keys, 20_000)]
        for x in got:
            assert np.all((x >= v[0].min() * (1 - 2.0 ** -7)) & (x <= v[0].max() * (1 + 2.0 ** -7)))


@pytest.mark.parametrize("fmt", ["bf16", "f16", "mxfp4"])
def test_fp32_queries_at_the_ends_of_their_range(gpu, fmt):
    """fp32 queries from fp32's smallest values to 2^126, over keys that keep the scores finite."""
    ud, d = gpu, 64
    for q_log, k_log in ((100, 0), (111, -10), (118, -14), (125, -20)):
        c, q = _huge(ud, fmt, "f32", d, q_log, k_log)
        ranges = np.array([[0, 330], [0, 330], [3, 217], [150, 320], [50, 160], [99, 152]])
        want = ref.attention(q, c.k, c.v, np.zeros(6, int), ranges, 0, 2, c.most * 16)
        _check_huge(window(ud, c, q[None], ranges[None], 0, "f32"), want, "f32", P_STEP[fmt, "f32"])
    rng = np.random.default_rng(100)
    c = Cache(ud, rng, fmt, [500], 2, d)
    for q_log in (-4, -30, -100, -120, -140):
        q = ref.rounded(rng.standard_normal((2, 4, d)) * 2.0 ** q_log, "f32")
        ranges = np.array([[0, 500], [20, 431]])
        want = ref.attention(q, c.k, c.v, np.zeros(2, int), ranges, 0, 2, c.most * 16)
        close(window(ud, c, q[None], ranges[None], 0, "f32"), want, c, d, "f32", P_STEP[fmt, "f32"])


def test_the_most_sequences(gpu):
    """65,535 sequences of one key each, in both attentions and the append: every row is its own key's value."""
    ud, rng, n, d = gpu, np.random.default_rng(101), 65_535, 64
    table = rng.permutation(n)[:, None].astype(np.int32)
    k, v, q = (ref.to_bits(rng.standard_normal((n, d)), "bf16") for _ in range(3))
    kp, vp, out = ud.DeviceBuffer(n * 16 * d * 2), ud.DeviceBuffer(n * 16 * d * 2), ud.DeviceBuffer(n * d * 2)
    bt, pos, qd = _dev(ud, table), _dev(ud, np.full(n, 5, np.int32)), _dev(ud, q)
    ud.qk_norm_rope_append(None, _dev(ud, k), _dev(ud, v), None, kp, vp, n, bt, n, 1, pos, n, 0, 1, d)
    ranges, start = _dev(ud, np.tile(np.array([5, 6], np.int32), (n, 1))), _dev(ud, np.arange(n + 1, dtype=np.int32))
    assert ud.gqa_window_workspace_bytes(n, 1, 1, 1, d, 0, 1) == ud.gqa_prefill_workspace_bytes(n, n, 1, 1, 1, d, 0, 1) == 0
    ud.gqa_window_attention_paged(qd, kp, vp, n, bt, 1, ranges, 0, out, n, 1, 1, 1, d, 1, None, dtype="bf16")
    ud.synchronize()
    np.testing.assert_array_equal(out.download((n, d), np.uint16), v)
    out = _dev(ud, np.zeros((n, d), np.uint16))
    ud.gqa_prefill_paged(qd, kp, vp, n, bt, 1, start, ranges, 0, out, n, n, 1, 1, 1, d, 1, None)
    ud.synchronize()
    np.testing.assert_array_equal(out.download((n, d), np.uint16), v)


def _prompt_calls(ud, fmt, dtype, span):
    """A ragged batch of prompts, and the call over given buffers."""
    rng, hq, hkv, d, new, past = np.random.default_rng(102), 8, 2, 128, [90, 1, 37], [700, 300, 0]
    rows, start = sum(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    c = Cache(ud, rng, fmt, [a + b for a, b in zip(new, past)], hkv, d)
    ranges = causal(new, past, 200)
    qs, rd, need = _dev(ud, start), _dev(ud, ranges.astype(np.int32)), ud.gqa_prefill_workspace_bytes(3, rows, 90, hq, hkv, d, 4, span)

    def call(q, out, ws, stream):
        ud.gqa_prefill_paged(q, c.kp, c.vp, c.num, c.bt, c.most, qs, rd, 4, out, 3, rows, 90, hq, hkv, d, span, ws, dtype=dtype, kv_format=fmt,
                             hip_stream=stream)

    def fresh():
        q = ref.rounded(rng.standard_normal((rows, hq, d)), dtype)
        return q, ref.to_bits(q, dtype).reshape(rows, -1)
    expect = lambda q: prefill(ud, c, q, start, ranges, 4, dtype, span=span)  # noqa: E731
    read = lambda out: ref.from_bits(out.download((rows, hq, d), np.uint16), dtype)  # noqa: E731
    return call, fresh, expect, read, need, rows * hq * d * 2


@pytest.mark.parametrize("fmt,dtype,span", [("bf16", "bf16", 300), ("mxfp4", "f16", 20_000), ("f16", "f16", 20_000)])
def test_prompts_in_a_graph(gpu, fmt, dtype, span):
    """Captured once and replayed over new queries, eager calls between: the same bits every time."""
    ud, stream = gpu, gpu.HipStream()
    call, fresh, expect, read, need, size = _prompt_calls(ud, fmt, dtype, span)
    assert (need > 0) == (span > 1000)
    qd, out, ws = ud.DeviceBuffer(size), ud.DeviceBuffer(size), ud.DeviceBuffer(need) if need else None
    graph = None
    for _ in range(4):
        q, bits = fresh()
        want = expect(q)
        qd.upload(bits)
        ud.synchronize()
        if graph is None:
            with ud.Graph.capture(stream) as graph:
                call(qd, out, ws, stream)
        graph.launch(stream)
        stream.synchronize()
        np.testing.assert_array_equal(read(out), want)


def test_prompts_on_two_streams(gpu):
    ud, streams = gpu, [gpu.HipStream() for _ in range(2)]
    call, fresh, expect, read, need, size = _prompt_calls(ud, "mxfp4", "bf16", 20_000)
    q = [fresh() for _ in streams]
    want = [expect(x) for x, _ in q]
    buf = [(_dev(ud, bits), ud.DeviceBuffer(size), ud.DeviceBuffer(need)) for _, bits in q]
    ud.synchronize()
    for _ in range(20):
        for s, (qd, out, ws) in zip(streams, buf):
            call(qd, out, ws, s)
    ud.synchronize()
    for (_, out, _), w in zip(buf, want):
        np.testing.assert_array_equal(read(out), w)
