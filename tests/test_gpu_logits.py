"""GPU parity of ud_logits_process with its float64 form (layer_ref.py): vocabularies of one token to 200,000, histories,
biases, grammar masks, and the greedy token of what comes out."""
import numpy as np
import pytest

import layer_ref as ref

pytestmark = pytest.mark.gpu


def dev(ud, a):
    return None if a is None else ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def process(ud, x, dtype, tokens=None, ranges=None, penalties=None, biases=None, mask=None, mask_rows=None, pad=(0, 0), in_place=False,
            choose=True, mask_pad=0, hip_stream=None):
    """x [n, V] float64; biases (ids, values, ranges); mask bool [masks, V].  (out, token), and what lies behind them is checked."""
    n, V = x.shape
    bits = ref.stored(x, dtype)[0] if dtype != "f32" else x.astype(np.float32)
    src = np.full((n, V + pad[0]), 7, bits.dtype)
    src[:, :V] = bits
    ind = dev(ud, src)
    old = V + (pad[0] if in_place else pad[1])
    outd = ind if in_place else dev(ud, np.full((n, old), 7, np.float32))
    tokend = dev(ud, np.full(n + 1, 55, np.int32)) if choose else None
    words = None
    if mask is not None:
        words = np.full((len(mask), -(-V // 32) + mask_pad), 0xFFFFFFFF, np.uint32)
        words[:, :-(-V // 32)] = ref.mask_words(mask)
    ws = ud.DeviceBuffer(max(8, ud.logits_workspace_bytes(n, V))) if choose else None
    b = biases or (None, None, None)
    ud.logits_process(ind, outd, n, V, token=tokend, tokens=dev(ud, tokens), n_tokens=0 if tokens is None else len(tokens),
                      ranges=dev(ud, ranges), penalties=dev(ud, penalties), bias_ids=dev(ud, b[0]), bias_values=dev(ud, b[1]),
                      n_biases=0 if b[0] is None else len(b[0]), bias_ranges=dev(ud, b[2]), mask=dev(ud, words),
                      n_masks=0 if mask is None else len(mask), mask_rows=dev(ud, mask_rows), workspace=ws, dtype=dtype,
                      ld=V + pad[0], out_ld=old, mask_ld=None if mask is None else words.shape[1])
    ud.synchronize()
    out = outd.download((n, old))
    assert np.all(out[:, V:] == 7)
    token = None
    if choose:
        token = tokend.download(n + 1, np.int32)
        assert token[-1] == 55
        token = token[:-1]
    return out[:, :V].astype(np.float64), token


def check(ud, rng, n, V, dtype, history=300, biases=20, masks="some", penalties=True, **kw):
    x = ref.stored(3 * rng.standard_normal((n, V)), dtype)[1]
    tokens = ranges = pen = b = mask = mask_rows = None
    if history:
        lens = rng.integers(0, history, n)
        lens[0] = history
        at = np.concatenate([[0], np.cumsum(lens)])
        tokens = np.minimum(V - 1, (V * rng.random(at[-1]) ** 3)).astype(np.int32)
        ranges = np.stack([at[:-1], at[:-1] + (lens * rng.random(n)).astype(int), at[1:]], 1).astype(np.int32)
        pen = (np.array([1, 0, 0]) + rng.random((n, 3)) * [0.5, 1, 0.5]).astype(np.float32)
    if biases:
        ids = rng.integers(0, V, n * biases).astype(np.int32)
        b = (ids, (2 * rng.standard_normal(n * biases)).astype(np.float32),
             np.stack([np.arange(n) * biases, (np.arange(n) + 1) * biases], 1).astype(np.int32))
    if masks:
        mask = rng.random((n, V)) < rng.choice([0.0, 0.01, 0.5, 1.0], (n, 1))
        mask_rows = rng.integers(-1, n, n).astype(np.int32)
    out, token = process(ud, x, dtype, tokens, ranges, pen, b, mask, mask_rows, **kw)
    want, mag = ref.logits_out(x, tokens, ranges, pen, None if b is None else [(b[0][lo:hi], b[1][lo:hi]) for lo, hi in b[2]],
                               None if mask is None else [mask[m] if m >= 0 else None for m in mask_rows])
    compare(out, want, mag)
    if token is not None:
        np.testing.assert_array_equal(token, ref.chosen(out))


def compare(out, want, mag):
    np.testing.assert_array_equal(np.isnan(out), np.isnan(want))
    far = ~np.isfinite(want) & ~np.isnan(want)
    np.testing.assert_array_equal(out[far], want[far])
    fine = np.isfinite(want)
    # the repetition's reciprocal and product, the count's product with presence, the difference, the bias: five roundings of what is
    # at most mag
    assert np.all(np.abs(out - want)[fine] <= 5.05 * ref.STEP32 * mag[fine])


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 31, 33, 1025, 2047, 2048, 2049, 4097, 8191, 8193, 32001, 131072, 200001])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_vocabularies(gpu, dtype, V):
    rng = np.random.default_rng([V, len(dtype)])
    check(gpu, rng, 1, V, dtype)
    check(gpu, rng, 5, V, dtype, pad=(1, 3), mask_pad=2)


@pytest.mark.parametrize("n,V", [(300, 1025), (70, 20000), (40, 131073), (600, 4000)])
def test_batches(gpu, n, V):
    """Each number of pieces per thread."""
    rng = np.random.default_rng(n)
    check(gpu, rng, n, V, "bf16", history=200)
    check(gpu, rng, n, V, "f32", history=50, biases=3, in_place=True, pad=(2, 0))


@pytest.mark.parametrize("history,biases,masks", [(0, 0, None), (50, 0, None), (0, 9, None), (0, 0, "some"), (5000, 0, None), (0, 3000, "some")])
def test_parts_alone(gpu, history, biases, masks):
    rng = np.random.default_rng([history, biases])
    check(gpu, rng, 4, 5000, "f32", history=history, biases=biases, masks=masks)
    check(gpu, rng, 4, 5000, "f16", history=history, biases=biases, masks=masks, choose=False)


def test_equal_logits(gpu):
    """The lowest of equal ones, over segments and threads; -0 and 0 are equal."""
    rng = np.random.default_rng(1)
    x = np.zeros((6, 140000))
    x[1, 100:] = -0.0
    x[1, :100] = -1
    x[2] = -np.inf
    x[2, 139999] = -2.0 ** 127
    for i in range(3, 6):
        x[i, rng.integers(0, 140000, 5)] = 2.5
    out, token = process(gpu, x, "f32")
    np.testing.assert_array_equal(out, x)
    np.testing.assert_array_equal(token, ref.chosen(x))
    assert token[0] == 0 and token[1] == 100 and token[2] == 139999


def test_no_numbers_and_nothing_left(gpu):
    V = 3000
    x = np.zeros((7, V))
    x[0] = np.nan
    x[1, 5], x[1, 9] = np.nan, 1
    x[2, 7] = np.inf
    x[3] = -np.inf
    x[4, 2999], x[4, 3] = np.inf, np.nan
    x[5], x[6] = np.nan, -3.4e38
    mask = np.ones((7, V), bool)
    mask[4, 2999] = False
    mask[5, 10:] = False
    mask[6] = False
    out, token = process(gpu, x, "f32", mask=mask)
    want = np.where(mask, x, -np.inf)
    np.testing.assert_array_equal(out, want.astype(np.float32))
    assert list(token) == [-1, 9, 7, -1, 0, -1, -1]


def test_ranges_and_ids_outside(gpu):
    """Ranges are cut to the arrays, ids outside the vocabulary are padding, a bias listed twice counts once (the last), rows
    share histories and lists, an empty or backward range is none, the boundary may lie outside the range."""
    V, rng = 2500, np.random.default_rng(2)
    x = rng.standard_normal((8, V))
    x = x.astype(np.float32).astype(np.float64)
    tokens = np.array([5, 5, 2499, -1, 2500, 2 ** 31 - 1, 7, 5, 2047, 2048, -2 ** 31], np.int32)
    ranges = np.array([[-5, 2, 11], [0, 0, 99], [3, 1, 7], [6, 99, 11], [4, 4, 4], [9, 5, 2], [0, 11, 11], [2 ** 31 - 1, 0, 2 ** 31 - 1]], np.int32)
    pen = np.tile(np.array([[1.25, 0.5, 0.25]], np.float32), (8, 1))
    ids = np.array([3, 2499, 3, -1, 2500, 3, 9], np.int32)
    vals = np.array([1, 2, 4, 8, 16, 32, -np.inf], np.float32)
    br = np.array([[0, 7], [0, 5], [2, 4], [-3, 1], [5, 99], [4, 4], [6, 2], [2 ** 31 - 1, 2 ** 31 - 1]], np.int32)
    out, token = process(gpu, x, "f32", tokens, ranges, pen, (ids, vals, br))
    cut = [(ids[max(0, lo):min(7, max(hi, 0))], vals[max(0, lo):min(7, max(hi, 0))]) if hi > lo else ([], []) for lo, hi in br]
    want, mag = ref.logits_out(x, tokens, ranges, pen, cut, None)
    compare(out, want, mag)
    np.testing.assert_array_equal(token, ref.chosen(out))


def test_shared_masks(gpu):
    V, rng = 9000, np.random.default_rng(4)
    x = rng.standard_normal((5, V)).astype(np.float32).astype(np.float64)
    mask = rng.random((2, V)) < 0.3
    rows = np.array([1, -1, 0, 1, 2], np.int32)                          # 2: outside, no mask
    out, token = process(gpu, x, "f32", mask=mask, mask_rows=rows)
    want = np.stack([x[i] if m in (-1, 2) else np.where(mask[m], x[i], -np.inf) for i, m in enumerate(rows)])
    np.testing.assert_array_equal(out, want)
    np.testing.assert_array_equal(token, ref.chosen(want))


def test_long_histories(gpu):
    """100,000 tokens, one of them 60,000 times."""
    V, rng = 4100, np.random.default_rng(6)
    x = rng.standard_normal((2, V)).astype(np.float32).astype(np.float64)
    tokens = rng.integers(0, V, 100000).astype(np.int32)
    tokens[rng.permutation(100000)[:60000]] = 4099
    ranges = np.array([[0, 0, 100000], [1, 50003, 99999]], np.int32)
    pen = np.array([[1.1, 0.1, 0.001], [0.9, -0.2, -0.002]], np.float32)
    out, token = process(gpu, x, "f32", tokens, ranges, pen)
    want, mag = ref.logits_out(x, tokens, ranges, pen, None, None)
    compare(out, want, mag)
    np.testing.assert_array_equal(token, ref.chosen(out))


@pytest.mark.parametrize("history,biases", [(65535, 32767), (65536, 10), (70000, 0), (10, 32768), (0, 40000), (70000, 40000)])
def test_lists_of_any_length(gpu, history, biases):
    """Lists that fit one word a token, just do not, and far from it."""
    rng = np.random.default_rng([history, biases])
    check(gpu, rng, 2, 9001, "f32", history=history, biases=biases)
    check(gpu, rng, 1, 300, "bf16", history=history, biases=biases, masks=None)


@pytest.mark.parametrize("n,V", [(2, 100001), (9, 60000), (20, 120001), (130, 32769), (260, 30000)])
def test_segments(gpu, n, V):
    """Each size of segment."""
    check(gpu, np.random.default_rng([n, V]), n, V, "f16", history=400)


def test_far_penalties(gpu):
    """Quotients past fp32's range, infinities and NaN under penalties and biases."""
    x = np.array([[3e38, -3e38, np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-38, 5.0]]).astype(np.float32).astype(np.float64)
    tokens = np.arange(9, dtype=np.int32)
    out, token = process(gpu, x, "f32", tokens, np.array([[0, 9, 9]], np.int32), np.array([[0.5, 9, 9]], np.float32))
    with np.errstate(over="ignore"):
        want = np.where(x > 0, x / 0.5, x * 0.5).astype(np.float32)
    np.testing.assert_array_equal(out, want)
    assert token[0] == 0                                   # the first of two infinities
    out, token = process(gpu, x, "f32", tokens, np.array([[0, 0, 9]], np.int32), np.array([[1, 1, 1]], np.float32),
                         (np.array([2, 3, 8], np.int32), np.array([-np.inf, np.inf, 1], np.float32), np.array([[0, 3]], np.int32)))
    assert np.all(np.isnan(out[0, 2:5])) and out[0, 8] == 4 and token[0] == 0


def test_no_rows(gpu):
    b = dev(gpu, np.zeros(64, np.float32))
    gpu.logits_process(b, b, 0, 4)
