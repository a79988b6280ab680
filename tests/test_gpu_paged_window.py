"""GPU parity of the windowed attention calls (ud_gqa_window_attention_paged, ud_gqa_prefill_paged) with their float64 form
(paged_ref.py), elementwise at tolerances counted from the roundings: page formats and query types, groups, lengths around
page and chunk borders, windows and sinks, empty rows, values that are no numbers where they are masked, pages given back,
pools past 4 GiB, splits; then the operators together, as a decoder runs them, eagerly and from replayed graphs."""
import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("mxfp4", "bf16"), ("mxfp4", "f16"), ("mxfp4", "f32")]
# half a step of a probability's rounding: 8 significant bits of bf16, 11 of half, 16 of two terms of bf16; fp32: three
# terms of bf16 (24 bits), two of half (22)
P_STEP = {("bf16", "bf16"): 2.0 ** -8, ("f16", "f16"): 2.0 ** -11, ("mxfp4", "bf16"): 2.0 ** -8, ("mxfp4", "f16"): 2.0 ** -16,
          ("bf16", "f32"): 2.0 ** -24, ("f16", "f32"): 2.0 ** -22, ("mxfp4", "f32"): 2.0 ** -24}
PROMPT_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def _dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


class Cache:
    """A paged cache of random (or given) keys and values, on the host and the device."""

    def __init__(self, ud, rng, fmt, lens, hkv, d, keep=None, k=None, v=None):
        self.fmt, self.lens, self.hkv, self.d = fmt, lens, hkv, d
        self.k = k or [ref.held(rng.standard_normal((L, hkv, d)), fmt) for L in lens]
        self.v = v or [ref.held(rng.standard_normal((L, hkv, d)), fmt) for L in lens]
        self.table, self.num = ref.assign_pages(rng, lens, keep=keep)
        pools = [ref.new_pool(fmt, self.num, hkv, d) for _ in range(2)]
        ref.fill(pools[0], self.table, fmt, d, self.k, self.num)
        ref.fill(pools[1], self.table, fmt, d, self.v, self.num)
        self.kp, self.vp, self.bt = _dev(ud, pools[0]), _dev(ud, pools[1]), _dev(ud, self.table)
        self.most = self.table.shape[1]

    def held_keys(self, i):
        page = self.table[i, np.arange(self.most * 16) // 16]
        return (page >= 0) & (page < self.num)


def window(ud, c, q, ranges, sinks, dtype, span=None, stream=None):
    """q [n, M, hq, d] float64 values of dtype -> [n, M, hq, d]."""
    n, M, hq, d = q.shape
    live = ranges[ranges[..., 0] < ranges[..., 1]]
    if span is None:
        span = max([1] + [int(r[:, 1][ok].max() - r[:, 0][ok].min()) for r in ranges for ok in [r[:, 0] < r[:, 1]] if ok.any()])
    need = ud.gqa_window_workspace_bytes(n, M, hq, c.hkv, d, sinks, span)
    ws = _dev(ud, np.full(need, 0xFF, np.uint8)) if need else None
    out = _dev(ud, np.full((n * M, hq * d), 0x7FFF, np.uint16) if dtype != "f32" else np.full((n * M, hq * d), np.nan, np.float32))
    qd, rd = _dev(ud, ref.to_bits(q, dtype).reshape(n * M, -1)), _dev(ud, ranges.astype(np.int32))
    ud.gqa_window_attention_paged(qd, c.kp, c.vp, c.num, c.bt, c.most, rd, sinks, out, n, M, hq, c.hkv, d, span, ws, dtype=dtype,
                                  kv_format=c.fmt, hip_stream=stream)
    ud.synchronize()
    return ref.from_bits(out.download((n, M, hq, d), np.float32 if dtype == "f32" else np.uint16), dtype)


def close(got, want, c, d, dtype, p_step):
    out, mag, top, dot, count = want
    got = got.reshape(out.shape)
    tol = ref.attention_tolerance(out, mag, top, dot, count, d, dtype, p_step)
    if dtype == "f16":
        tol = tol + 2.0 ** -25                          # an output below half's normal range: half its smallest step
    if dtype == "f16" or c.fmt == "f16":
        # a probability below half's normal range is off by half the smallest step, 2^-25 of 2^7 times it; their sum is 1 or more
        most = max([np.abs(x[np.isfinite(x)]).max(initial=0) for x in c.v])
        tol = tol + (count * 2.0 ** -32 * most)[:, None, None]
    off = np.abs(got - out)
    assert np.all(off <= tol), "worst %.3g of its tolerance at %s" % (np.nanmax(off / tol), np.unravel_index(np.nanargmax(off / tol), off.shape))
    assert np.all(got[count == 0] == 0)


def check_window(ud, rng, fmt, dtype, hq, hkv, d, lens, M, win, sinks, empty=(), span=None, give_back=False):
    n = len(lens)
    ends = np.array([[max(0, L - M + 1 + m) for m in range(M)] for L in lens])
    ranges = np.stack([np.maximum(0, ends - win) if win else np.zeros_like(ends), ends], -1)
    for i, m in empty:
        ranges[i, m] = [5, 5 - m]
    keep = None
    if give_back:
        lows = [min([r[0] for r in ranges[i] if r[0] < r[1]] or [0]) for i in range(n)]
        keep = lambda i, b: b * 16 < min(sinks, lows[i]) or b * 16 + 16 > lows[i]  # noqa: E731
    c = Cache(ud, rng, fmt, lens, hkv, d, keep=keep)
    q = ref.rounded(rng.standard_normal((n, M, hq, d)) * 1.5, dtype)
    got = window(ud, c, q, ranges, sinks, dtype, span=span)
    want = ref.attention(q.reshape(n * M, hq, d), c.k, c.v, np.repeat(np.arange(n), M), ranges.reshape(-1, 2), sinks, hkv, c.most * 16)
    close(got, want, c, d, dtype, P_STEP[fmt, dtype])


LENS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 129, 300, 700]


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (7, 1, 128), (8, 1, 64), (3, 3, 64)])
def test_window_types_and_heads(gpu, fmt, dtype, hq, hkv, d):
    rng = np.random.default_rng([hq, d, len(fmt), len(dtype)])
    check_window(gpu, rng, fmt, dtype, hq, hkv, d, LENS, 1, 0, 0)
    check_window(gpu, rng, fmt, dtype, hq, hkv, d, LENS, 3, 50, 5, empty=[(2, 0), (9, 1), (4, 0), (4, 1), (4, 2)], give_back=True)


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("group,M,d", [(1, 1, 128), (16, 1, 64), (8, 8, 128), (2, 8, 64), (5, 4, 128), (7, 5, 64), (64, 1, 128)])
def test_window_row_tiles(gpu, fmt, dtype, group, M, d):
    """1 .. 64 query rows per kv head, whole and partly filled tiles of 16."""
    rng = np.random.default_rng([group, M, d, len(fmt), len(dtype)])
    check_window(gpu, rng, fmt, dtype, 2 * group, 2, d, [9, 100, 333], M, 70, 20, give_back=True)


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f32"), ("mxfp4", "f32")])
@pytest.mark.parametrize("win,sinks", [(1, 0), (1, 1), (16, 16), (17, 1), (100, 64), (1000, 3), (2000, 5000), (0, 7)])
def test_windows_and_sinks(gpu, fmt, dtype, win, sinks):
    """Windows of one key up to more than the context, sinks that meet or overlap the window's first page."""
    rng = np.random.default_rng([win, sinks, len(fmt)])
    check_window(gpu, rng, fmt, dtype, 4, 1, 128, [1, 16, 17, 100, 950, 1500], 1, win, sinks, give_back=True)


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f16"), ("mxfp4", "f32")])
def test_long_context_many_splits(gpu, fmt, dtype):
    """One sequence over the whole chip (the most splits), and a span that the caller gave too small."""
    rng = np.random.default_rng(11)
    for span in (None, 300, 1):
        check_window(gpu, rng, fmt, dtype, 4, 1, 64, [12_345, 77], 1, 0, 0, span=span)


@pytest.mark.parametrize("fmt", ["bf16", "f16", "mxfp4"])
def test_window_masked_values_are_not_seen(gpu, fmt):
    """NaN and infinities in keys and values behind the range, between the sinks and the window, and where only the last
    of the queries may look: every other row is as without them."""
    ud, rng, hq, hkv, d, M = gpu, np.random.default_rng(12), 4, 2, 64, 4
    lens = [200, 37, 90]
    c0 = Cache(ud, np.random.default_rng(13), fmt, lens, hkv, d)
    k, v = [x.copy() for x in c0.k], [x.copy() for x in c0.v]
    ranges = np.array([[[L - 30 - m, L - 10 + m] for m in range(M)] for L in lens])
    ranges[1, 1] = [9, 9]
    bad = [np.nan, np.inf, -np.inf, np.nan]
    for i, L in enumerate(lens):
        for x in (k[i], v[i]):
            x[L - 10 + M - 1:] = bad[i]                 # behind every range
            x[6:L - 30 - M + 1] = bad[i + 1]            # between sinks and windows (none for the short one)
    only_last = lens[0] - 10 + M - 2                    # seen by the last query of sequence 0 alone
    for x in (k[0], v[0]):
        x[only_last] = np.nan
    q = ref.rounded(rng.standard_normal((3, M, hq, d)), "f32")
    for dtype in ("f32", "bf16" if fmt != "f16" else "f16"):
        qq = ref.rounded(q, dtype)
        clean = window(ud, c0, qq, ranges, 6, dtype)
        c1 = Cache(ud, np.random.default_rng(13), fmt, lens, hkv, d, k=k, v=v)
        got = window(ud, c1, qq, ranges, 6, dtype)
        assert np.all(np.isnan(got[0, M - 1]))
        got[0, M - 1] = clean[0, M - 1]
        np.testing.assert_array_equal(got, clean)


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("d,hkv,lens", [(128, 16, [1, 16, 33] + list(range(40, 300, 17))), (64, 90, [2100, 64, 700])])
def test_window_more_than_a_round_of_workgroups(gpu, fmt, dtype, d, hkv, lens):
    """More sequences times kv heads than CUs: short ones (workgroups of four waves), and one long enough for eight."""
    assert len(lens) * hkv > 256
    rng = np.random.default_rng([71, d, len(fmt), len(dtype)])
    check_window(gpu, rng, fmt, dtype, hkv, hkv, d, lens, 2, 0, 0, empty=[(1, 1)])
    check_window(gpu, rng, fmt, dtype, hkv, hkv, d, lens, 1, 100, 5, give_back=True)


@pytest.mark.parametrize("fmt,dtype", TYPES)
@pytest.mark.parametrize("n,hkv,M", [(60, 5, 1), (64, 5, 3), (2, 200, 1), (33, 8, 2)])
def test_window_batches_taken_by_length(gpu, fmt, dtype, n, hkv, M):
    """Long ragged batches of up to 64 sequences, equal lengths and rows that see nothing among them."""
    rng = np.random.default_rng([74, n, M, len(fmt), len(dtype)])
    lens = [2100, 17] + [int(x) for x in rng.choice([5, 64, 64, 130, 300, 301], n - 2)]
    empty = [(i, m) for i in range(0, n, 7) for m in range(M) if i] + [(1, M - 1)]
    check_window(gpu, rng, fmt, dtype, 2 * hkv, hkv, 64, lens, M, 0, 0, empty=empty)


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f32"), ("mxfp4", "bf16")])
def test_window_masked_values_in_many_workgroups(gpu, fmt, dtype):
    """NaN and infinities behind the range and between sinks and window, on more units than CUs: nothing changes; in a key and a
    value that is seen: that head's rows alone are NaN."""
    ud, rng, hkv, d = gpu, np.random.default_rng(72), 100, 64
    lens = [150, 40, 97]
    c0 = Cache(ud, np.random.default_rng(73), fmt, lens, hkv, d)
    ranges = np.array([[[L - 31, L - 10]] for L in lens])
    q = ref.rounded(rng.standard_normal((3, 1, hkv, d)), dtype)
    clean = window(ud, c0, q, ranges, 4, dtype)
    k, v = [x.copy() for x in c0.k], [x.copy() for x in c0.v]
    for i, L in enumerate(lens):
        for x in (k[i], v[i]):
            x[L - 10:] = (np.nan, np.inf, -np.inf)[i]
            x[4:L - 31] = (np.inf, np.nan, np.nan)[i]
    c1 = Cache(ud, np.random.default_rng(73), fmt, lens, hkv, d, k=k, v=v)
    np.testing.assert_array_equal(window(ud, c1, q, ranges, 4, dtype), clean)
    v[2][80, 55] = np.nan
    k[0][135, 7] = np.nan
    c2 = Cache(ud, np.random.default_rng(73), fmt, lens, hkv, d, k=k, v=v)
    got = window(ud, c2, q, ranges, 4, dtype)
    assert np.all(np.isnan(got[2, 0, 55])) and np.all(np.isnan(got[0, 0, 7]))
    got[2, 0, 55], got[0, 0, 7] = clean[2, 0, 55], clean[0, 0, 7]
    np.testing.assert_array_equal(got, clean)


def test_window_pages_that_are_not_held(gpu):
    """A block-table entry outside the pool inside the range: its keys are not there."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(14), 4, 2, 128
    for fmt, dtype in (("bf16", "bf16"), ("mxfp4", "f32")):
        c = Cache(ud, rng, fmt, [100, 40, 16], hkv, d, keep=lambda i, b: (i, b) not in ((0, 2), (0, 6), (2, 0)))
        q = ref.rounded(rng.standard_normal((3, 1, hq, d)), dtype)
        ranges = np.array([[[0, 100]], [[3, 40]], [[0, 16]]])
        got = window(ud, c, q, ranges, 0, dtype)
        want = ref.attention(q[:, 0], c.k, c.v, np.arange(3), ranges[:, 0], 0, hkv, c.most * 16, held_keys=c.held_keys)
        close(got, want, c, d, dtype, P_STEP[fmt, dtype])


def test_ranges_are_cut_to_the_table(gpu):
    ud, rng = gpu, np.random.default_rng(15)
    c = Cache(ud, rng, "bf16", [48, 48], 1, 64)
    q = ref.rounded(rng.standard_normal((2, 1, 2, 64)), "bf16")
    wide = window(ud, c, q, np.array([[[-2 ** 31, 2 ** 31 - 1]], [[-5, 48]]]), 2 ** 31 - 1, "bf16", span=48)
    np.testing.assert_array_equal(wide, window(ud, c, q, np.array([[[0, 48]], [[0, 48]]]), 0, "bf16", span=48))


@pytest.mark.parametrize("fmt", ["bf16", "mxfp4"])
def test_pool_past_4_gib(gpu, fmt):
    """Pages whose byte offsets pass 32 bits, written by the append, read by both attentions and the read-back."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(16), 8, 8, 128
    each = ud.kv_page_bytes(hkv, d, fmt)
    num = (5 << 30) // each
    kp, vp = ud.DeviceBuffer(num * each), ud.DeviceBuffer(num * each)
    pages = np.array([[num - 1, 0, num - 2, (1 << 32) // each + 1]], np.int32)
    x = ref.rounded(rng.standard_normal((50, hq + 2 * hkv, d)), "bf16")
    pos, seqs = np.arange(50, dtype=np.int32), np.zeros(50, np.int32)
    bits = ref.to_bits(x, "bf16").reshape(50, -1)
    cut = [_dev(ud, bits[:, a * d:b * d]) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
    out, bt, pd, sd = ud.DeviceBuffer(50 * hq * d * 2), _dev(ud, pages), _dev(ud, pos), _dev(ud, seqs)
    ud.qk_norm_rope_append(cut[0], cut[1], cut[2], out, kp, vp, num, bt, 1, 4, pd, 50, hq, hkv, d, seqs=sd, kv_format=fmt)
    back = [ud.DeviceBuffer(50 * hkv * d * 4) for _ in range(2)]
    ud.paged_kv_read(kp, vp, num, bt, 1, 4, pd, back[0], back[1], 50, hkv, d, seqs=sd, dtype="f32", kv_format=fmt)
    ud.synchronize()
    k, v = ref.held(x[:, hq:hq + hkv], fmt), ref.held(x[:, hq + hkv:], fmt)
    np.testing.assert_array_equal(back[0].download((50, hkv, d)), k)
    np.testing.assert_array_equal(back[1].download((50, hkv, d)), v)
    c = type("C", (), dict(kp=kp, vp=vp, bt=bt, num=num, most=4, fmt=fmt, hkv=hkv))
    want = ref.attention(x[:, :hq], [k], [v], seqs, np.stack([0 * pos, pos + 1], -1), 0, hkv, 64)
    got = window(ud, c, x[49:, :hq][None], np.array([[[0, 50]]]), 0, "bf16")
    close(got, [w[49:] for w in want], c, d, "bf16", 2.0 ** -8)
    got = prefill(ud, c, x[:, :hq], [0, 50], np.stack([0 * pos, pos + 1], -1), 0, "bf16")
    close(got, want, c, d, "bf16", 2.0 ** -8)


# ---------------------------------------------------------------- prompts

def prefill(ud, c, q, start, ranges, sinks, dtype, span=None, most=None, rows=None, stream=None):
    rows, hq, d = q.shape
    start = np.asarray(start, np.int32)
    if span is None:
        span = 1
        for a, b in zip(start[:-1], start[1:]):
            r = ranges[a:b][ranges[a:b, 0] < ranges[a:b, 1]]
            if len(r):
                span = max(span, int(r[:, 1].max() - r[:, 0].min()))
    most = int(max(1, np.diff(start).max())) if most is None else most
    n = len(start) - 1
    need = ud.gqa_prefill_workspace_bytes(n, rows, most, hq, c.hkv, d, sinks, span)
    ws = _dev(ud, np.full(need, 0xFF, np.uint8)) if need else None
    out = _dev(ud, np.full((rows, hq * d), 0x1234, np.uint16))
    ud.gqa_prefill_paged(_dev(ud, ref.to_bits(q, dtype).reshape(rows, -1)), c.kp, c.vp, c.num, c.bt, c.most, _dev(ud, start),
                         _dev(ud, ranges.astype(np.int32)), sinks, out, n, rows, most, hq, c.hkv, d, span, ws, dtype=dtype,
                         kv_format=c.fmt, hip_stream=stream)
    ud.synchronize()
    return ref.from_bits(out.download((rows, hq, d), np.uint16), dtype)


def causal(new, past, win):
    ends = np.concatenate([p + 1 + np.arange(t) for t, p in zip(new, past)])
    return np.stack([np.maximum(0, ends - win) if win else 0 * ends, ends], -1)


PROMPTS = [("bf16", "bf16"), ("f16", "f16"), ("mxfp4", "bf16"), ("mxfp4", "f16")]


def check_prefill(ud, rng, fmt, dtype, hq, hkv, d, new, past, win, sinks, empty=(), give_back=False, **kw):
    ranges = causal(new, past, win)
    for r in empty:
        ranges[r] = [40, 3]
    start = np.concatenate([[0], np.cumsum(new)])
    keep = None
    if give_back:
        low = [max(0, p + 1 - win) if win else 0 for p in past]
        keep = lambda i, b: b * 16 < min(sinks, low[i]) or b * 16 + 16 > low[i]  # noqa: E731
    c = Cache(ud, rng, fmt, [max(1, t + p) for t, p in zip(new, past)], hkv, d, keep=keep)
    q = ref.rounded(rng.standard_normal((start[-1], hq, d)) * 1.5, dtype)
    got = prefill(ud, c, q, start, ranges, sinks, dtype, **kw)
    want = ref.attention(q, c.k, c.v, np.repeat(np.arange(len(new)), new), ranges, sinks, hkv, c.most * 16)
    # half queries on MXFP4: probabilities are rounded to half
    close(got, want, c, d, dtype, PROMPT_STEP[dtype])


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (7, 1, 128), (8, 1, 64), (2, 2, 64)])
def test_prefill_types_and_heads(gpu, fmt, dtype, hq, hkv, d):
    rng = np.random.default_rng([hq, d, len(fmt), len(dtype)])
    check_prefill(gpu, rng, fmt, dtype, hq, hkv, d, [1, 0, 65, 17, 130], [0, 5, 0, 100, 3], 0, 0)
    check_prefill(gpu, rng, fmt, dtype, hq, hkv, d, [64, 3, 150, 1], [0, 61, 200, 333], 50, 5, empty=[0, 66, 100], give_back=True)


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
def test_prefill_windows_sinks_and_splits(gpu, fmt, dtype):
    """Windows of one key up to more than the prompt; few rows over a long cache (keys split over workgroups)."""
    rng = np.random.default_rng(21)
    for win, sinks in [(1, 0), (1, 3), (16, 16), (33, 64), (500, 2000), (0, 9)]:
        check_prefill(gpu, rng, fmt, dtype, 4, 1, 64, [70, 200], [0, 40], win, sinks, give_back=True)
    check_prefill(gpu, rng, fmt, dtype, 4, 2, 128, [5, 19], [6000, 2048], 0, 0)
    check_prefill(gpu, rng, fmt, dtype, 4, 2, 128, [5, 19], [6000, 2048], 3000, 33, span=10, give_back=True)
    check_prefill(gpu, rng, fmt, dtype, 4, 2, 128, [9], [7000], 0, 0, empty=[2])


def test_prefill_general_ranges(gpu):
    """Ranges in any order: chunks that look ahead, rows that look far back beside rows that do not, rows without a key."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(22), 4, 2, 128
    for fmt, dtype in PROMPTS:
        c = Cache(ud, rng, fmt, [500, 333], hkv, d)
        lo = rng.integers(0, 330, 300)
        ranges = np.stack([lo, np.minimum(lo + rng.integers(-5, 200, 300), 333)], -1)
        q = ref.rounded(rng.standard_normal((300, hq, d)), dtype)
        got = prefill(ud, c, q, [0, 123, 300], ranges, 30, dtype, span=333)
        want = ref.attention(q, c.k, c.v, np.repeat([0, 1], [123, 177]), ranges, 30, hkv, c.most * 16)
        close(got, want, c, d, dtype, PROMPT_STEP[dtype])


@pytest.mark.parametrize("span", [100, 20000])
def test_prefill_rows_of_no_sequence(gpu, span):
    """Rows before the first, behind the last sequence, and past max_rows of one stay as they were; with splits too."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(23), 4, 2, 64
    c = Cache(ud, rng, "bf16", [90, 90], hkv, d)
    q = ref.rounded(rng.standard_normal((90, hq, d)), "bf16")
    ranges = np.stack([np.zeros(90, int), np.full(90, 90)], -1)
    need = ud.gqa_prefill_workspace_bytes(2, 90, 30, hq, hkv, d, 0, span)
    assert (need > 0) == (span > 1000)
    got = prefill(ud, c, q, [7, 30, 70], ranges, 0, "bf16", span=span, most=30)
    untouched = ref.from_bits(np.full(1, 0x1234, np.uint16), "bf16")[0]
    done = np.zeros(90, bool)
    done[7:60] = True
    assert np.all(got[~done] == untouched)
    want = ref.attention(q[done], c.k, c.v, np.repeat([0, 1], [23, 30]), ranges[done], 0, hkv, c.most * 16)
    close(got[done], want, c, d, "bf16", 2.0 ** -8)


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
def test_prefill_masked_values_are_not_seen(gpu, fmt, dtype):
    """A token whose key and value are no numbers, in the middle of a causal prompt: earlier rows are as without it."""
    ud, hq, hkv, d = gpu, 4, 2, 128
    c0 = Cache(ud, np.random.default_rng(31), fmt, [150, 60], hkv, d)
    k, v = [x.copy() for x in c0.k], [x.copy() for x in c0.v]
    k[0][100], v[0][100] = np.nan, np.nan
    v[1][30:] = np.inf
    k[1][30:] = np.nan
    c1 = Cache(ud, np.random.default_rng(31), fmt, [150, 60], hkv, d, k=k, v=v)
    ranges = causal([150, 60], [0, 0], 0)
    ranges[150:, 1] = np.minimum(ranges[150:, 1], 30)
    q = ref.rounded(np.random.default_rng(32).standard_normal((210, hq, d)), dtype)
    clean, got = (prefill(ud, c, q, [0, 150, 210], ranges, 0, dtype) for c in (c0, c1))
    assert np.all(np.isnan(got[100:150]))
    got[100:150] = clean[100:150]
    np.testing.assert_array_equal(got, clean)


def test_half_queries_saturate_large_fp4(gpu):
    """A block past half's range: MXFP4 4 x 2^14 reads as 65504 under half queries."""
    ud, hq, hkv, d = gpu, 1, 1, 64
    v = np.zeros((16, 1, d))
    v[:, 0, 0], v[:, 0, 1], v[:, 0, 32], v[:, 0, 33] = 60000, -60000, 5, 100
    c = Cache(ud, np.random.default_rng(33), "mxfp4", [16], hkv, d, k=[np.zeros((16, 1, d))], v=[v])
    got = prefill(ud, c, np.ones((1, hq, d)), [0, 1], np.array([[0, 16]]), 0, "f16")[0, 0]
    held = ref.held(v[0, 0], "mxfp4")
    assert held[0] == 65536 and got[0] == 65504 and got[1] == -65504
    np.testing.assert_array_equal(got[2:], held[2:])


def _ramp(rng, lens, hkv, d, fmt):
    """Keys whose scores with a query along e climb (sequence 0), fall (1) or jump about (2) by far more than a running
    maximum is allowed to lag behind."""
    e = rng.standard_normal(d)
    e /= np.linalg.norm(e)
    out = []
    for i, L in enumerate(lens):
        t = np.arange(L) / 16
        a = (t, -t, 40 * rng.standard_normal(L))[i % 3]
        out.append(ref.held(0.1 * rng.standard_normal((L, hkv, d)) + a[:, None, None] * e, fmt))
    return e, out


@pytest.mark.parametrize("fmt,dtype", TYPES)
def test_window_steep_scores(gpu, fmt, dtype):
    """Scores that climb by hundreds over the keys: the sums are rescaled again and again, most of the keys end at 0."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(61), 8, 2, 128
    lens = [1500, 900, 1200]
    e, k = _ramp(rng, lens, hkv, d, fmt)
    c = Cache(ud, rng, fmt, lens, hkv, d, k=k)
    q = ref.rounded(rng.standard_normal((3, 2, hq, d)) * 0.3 + 30 * e, dtype)
    ranges = np.array([[[0, L], [L // 3, L - 7]] for L in lens])
    got = window(ud, c, q, ranges, 3, dtype)
    want = ref.attention(q.reshape(6, hq, d), c.k, c.v, np.repeat(np.arange(3), 2), ranges.reshape(-1, 2), 3, hkv, c.most * 16)
    close(got, want, c, d, dtype, P_STEP[fmt, dtype])


@pytest.mark.parametrize("fmt,dtype", PROMPTS)
def test_prefill_steep_scores(gpu, fmt, dtype):
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(62), 4, 2, 64
    lens = [400, 300, 350]
    e, k = _ramp(rng, lens, hkv, d, fmt)
    c = Cache(ud, rng, fmt, lens, hkv, d, k=k)
    new, past = [150, 60, 130], [250, 240, 220]
    q = ref.rounded(rng.standard_normal((340, hq, d)) * 0.3 + 30 * e, dtype)
    ranges = causal(new, past, 0)
    got = prefill(ud, c, q, [0, 150, 210, 340], ranges, 0, dtype)
    want = ref.attention(q, c.k, c.v, np.repeat(np.arange(3), new), ranges, 0, hkv, c.most * 16)
    close(got, want, c, d, dtype, PROMPT_STEP[dtype])


@pytest.mark.parametrize("fmt,dtype", [("bf16", "bf16"), ("f16", "f32"), ("mxfp4", "f16"), ("mxfp4", "f32"), ("f16", "f16")])
def test_queries_that_are_no_numbers(gpu, fmt, dtype):
    """A NaN or an infinity in one query row makes that row NaN and no other, an empty range stays 0."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(63), 4, 2, 64
    c = Cache(ud, rng, fmt, [700, 40], hkv, d)
    q = ref.rounded(rng.standard_normal((2, 3, hq, d)), dtype)
    ranges = np.array([[[0, 700], [5, 690], [9, 9]], [[0, 40], [0, 1], [0, 39]]])
    clean = window(ud, c, q, ranges, 0, dtype)
    bad = q.copy()
    bad[0, 1, 2, 7], bad[1, 0, 0, :], bad[0, 2, 1, 3], bad[1, 1, 3, 5] = np.nan, np.nan, np.nan, np.inf
    got = window(ud, c, bad, ranges, 0, dtype)
    rows = np.zeros(got.shape[:3], bool)
    rows[0, 1, 2] = rows[1, 0, 0] = rows[1, 1, 3] = True
    assert np.all(np.isnan(got[rows]))
    np.testing.assert_array_equal(got[~rows], clean[~rows])
    assert np.all(got[0, 2] == 0)
    if dtype == "f32":
        return
    new = causal([130], [0], 0)
    q = ref.rounded(rng.standard_normal((130, hq, d)), dtype)
    clean = prefill(ud, c, q, [0, 130], new, 0, dtype)
    bad = q.copy()
    bad[77, 1, 0] = np.nan
    got = prefill(ud, c, bad, [0, 130], new, 0, dtype)
    assert np.all(np.isnan(got[77, 1]))
    got[77, 1] = clean[77, 1]
    np.testing.assert_array_equal(got, clean)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("fmt,dtype,d", [("mxfp4", "bf16", 128), ("bf16", "bf16", 64), ("f16", "f16", 128), ("mxfp4", "f16", 64)])
@pytest.mark.parametrize("graph", [False, True])
def test_decoder_runs_them_together(gpu, fmt, dtype, d, graph):
    """Two prompts in two pieces, then single tokens: norm, rotation and append, attention over window and sinks.  Queries
    are checked against float64, the attention against float64 over what the pages hold.  graph: each token's two calls are
    captured once and replayed (positions and ranges change in place), with eager calls between."""
    ud, rng, hq, hkv, win, sinks = gpu, np.random.default_rng(41), 8, 2, 48, 5
    piece, steps, n = [[30, 75], [33, 10]], 6, 2
    lens = [sum(p[i] for p in piece) + steps for i in range(n)]
    w = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)]
    inv = ud.rope_inv_freq(d)
    table, num = ref.assign_pages(rng, lens)
    kp, vp = (_dev(ud, ref.new_pool(fmt, num, hkv, d)) for _ in range(2))
    bt, qw, kw, iv = _dev(ud, table), _dev(ud, w[0]), _dev(ud, w[1]), _dev(ud, inv)
    most = table.shape[1]
    k, v = [np.zeros((L, hkv, d)) for L in lens], [np.zeros((L, hkv, d)) for L in lens]
    c = type("C", (), dict(kp=kp, vp=vp, bt=bt, num=num, most=most, fmt=fmt, hkv=hkv))
    stream = ud.HipStream()

    def rows(pos, seqs):
        """New projected rows; the expected queries, and keys and values noted."""
        x = ref.rounded(rng.standard_normal((len(pos), hq + 2 * hkv, d)), dtype)
        kk = ref.norm_rope(x[:, hq:hq + hkv], w[1], 1e-6, pos, inv)
        for t in range(len(pos)):
            k[seqs[t]][pos[t]] = ref.held(kk[t], fmt)
            v[seqs[t]][pos[t]] = ref.held(x[t, hq + hkv:], fmt)
        return x, ref.norm_rope(x[:, :hq], w[0], 1e-6, pos, inv)

    def compare(got, q, seqs, ranges):
        want = ref.attention(q, k, v, seqs, ranges, sinks, hkv, most * 16)
        p_step = P_STEP[fmt, dtype] if len(q) == n else PROMPT_STEP[dtype]
        # the operator's queries and 16-bit keys are rounded once more than float64's: a score is off by up to 2 half
        # steps of sum |q||k|, so numerator and sum of the softmax by that much each (rounded values are larger by at
        # most a half step: 1.02)
        _, mag, _, dot, _ = want
        extra = 2 * 2 * ref.HALF_STEP[dtype] * 1.02 * dot[..., None] * mag
        off = np.abs(got - want[0])
        assert np.all(off <= ref.attention_tolerance(*want, d, dtype, p_step) + extra), np.max(off)

    done = [0] * n
    for new in piece:
        pos = np.concatenate([done[i] + np.arange(new[i]) for i in range(n)])
        seqs = np.repeat(np.arange(n), new)
        x, q = rows(pos, seqs)
        src, out, r = _dev(ud, ref.to_bits(x, dtype).reshape(len(pos), -1)), ud.DeviceBuffer(len(pos) * hq * d * 2), len(pos)
        ld = (hq + 2 * hkv) * d
        at = lambda off: type("At", (), dict(ptr=src.ptr + off * 2))  # noqa: E731
        ranges = causal(new, done, win)
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        att = ud.DeviceBuffer(r * hq * d * 2)
        need = ud.gqa_prefill_workspace_bytes(n, r, max(new), hq, hkv, d, sinks, 200)
        ws = ud.DeviceBuffer(need) if need else None
        keep = _dev(ud, pos.astype(np.int32)), _dev(ud, seqs.astype(np.int32)), _dev(ud, start), _dev(ud, ranges.astype(np.int32))
        ud.qk_norm_rope_append(at(0), at(hq * d), at((hq + hkv) * d), out, kp, vp, num, bt, n, most, keep[0], r, hq, hkv, d, seqs=keep[1],
                               q_weight=qw, k_weight=kw, inv_freq=iv, dtype=dtype, kv_format=fmt, q_ld=ld, k_ld=ld, v_ld=ld, hip_stream=stream)
        ud.gqa_prefill_paged(out, kp, vp, num, bt, most, keep[2], keep[3], sinks, att, n, r, max(new), hq, hkv, d, 200, ws, dtype=dtype,
                             kv_format=fmt, hip_stream=stream)
        stream.synchronize()
        compare(ref.from_bits(att.download((r, hq, d), np.uint16), dtype), q, seqs, ranges)
        done = [a + b for a, b in zip(done, new)]

    src, out, att = (ud.DeviceBuffer(n * x * d * 2) for x in (hq + 2 * hkv, hq, hq))
    posd, rd = ud.DeviceBuffer(n * 4), ud.DeviceBuffer(n * 8)
    need = ud.gqa_window_workspace_bytes(n, 1, hq, hkv, d, sinks, 4000)
    ws, ld = ud.DeviceBuffer(need), (hq + 2 * hkv) * d

    def token():
        at = lambda off: type("At", (), dict(ptr=src.ptr + off * 2))  # noqa: E731
        ud.qk_norm_rope_append(at(0), at(hq * d), at((hq + hkv) * d), out, kp, vp, num, bt, n, most, posd, n, hq, hkv, d, q_weight=qw,
                               k_weight=kw, inv_freq=iv, dtype=dtype, kv_format=fmt, q_ld=ld, k_ld=ld, v_ld=ld, hip_stream=stream)
        ud.gqa_window_attention_paged(out, kp, vp, num, bt, most, rd, sinks, att, n, 1, hq, hkv, d, 4000, ws, dtype=dtype, kv_format=fmt,
                                      hip_stream=stream)

    captured = None
    for step in range(steps):
        pos = np.array(done)
        x, q = rows(pos, np.arange(n))
        ranges = causal([1] * n, done, win)
        src.upload(ref.to_bits(x, dtype))
        posd.upload(pos.astype(np.int32))
        rd.upload(ranges.astype(np.int32))
        ud.synchronize()
        if graph and captured is None:
            with ud.Graph.capture(stream) as captured:
                token()
        if captured is not None:
            captured.launch(stream)
        else:
            token()
        stream.synchronize()
        got = ref.from_bits(att.download((n, hq, d), np.uint16), dtype)
        compare(got, q, np.arange(n), ranges)
        if graph:                                       # an eager run of the same step between the replays
            token()
            stream.synchronize()
            np.testing.assert_array_equal(got, ref.from_bits(att.download((n, hq, d), np.uint16), dtype))
        done = [a + 1 for a in done]


def test_two_streams_at_once(gpu):
    """Calls on two streams, each with its own workspace, give what they give alone."""
    ud, rng, hq, hkv, d = gpu, np.random.default_rng(51), 8, 2, 128
    c = Cache(ud, rng, "mxfp4", [3000, 900], hkv, d)
    q = [ref.rounded(rng.standard_normal((2, 1, hq, d)), "bf16") for _ in range(2)]
    ranges = np.array([[[0, 3000]], [[100, 900]]])
    alone = [window(ud, c, x, ranges, 4, "bf16") for x in q]
    streams = [ud.HipStream() for _ in range(2)]
    need = ud.gqa_window_workspace_bytes(2, 1, hq, hkv, d, 4, 3000)
    assert need
    buf = [(_dev(ud, ref.to_bits(x, "bf16")), _dev(ud, ranges.astype(np.int32)), ud.DeviceBuffer(need), ud.DeviceBuffer(2 * hq * d * 2)) for x in q]
    ud.synchronize()
    for _ in range(20):
        for s, (qd, rd, ws, out) in zip(streams, buf):
            ud.gqa_window_attention_paged(qd, c.kp, c.vp, c.num, c.bt, c.most, rd, 4, out, 2, 1, hq, hkv, d, 3000, ws, dtype="bf16",
                                          kv_format="mxfp4", hip_stream=s)
    ud.synchronize()
    for a, (_, _, _, out) in zip(alone, buf):
        np.testing.assert_array_equal(a, ref.from_bits(out.download(a.shape, np.uint16), "bf16"))
