"""Plain float64 forms of the calls of include/ud_layer.h: the residual's addition and the norm, rows in 8 bits, the int8
product, logits under penalties, biases and masks.  numpy only; used by the tests of those calls."""
import numpy as np

from paged_ref import HALF_STEP, from_bits, to_bits  # noqa: F401

STEP32 = 2.0 ** -24                    # half a step of fp32, relative
TINY = 2.0 ** -126
# A half under 2^-14 is a multiple of 2^-24: a rounding is off by 2^-25 at most.
FLOOR = {"bf16": 0.0, "f16": 2.0 ** -25, "f32": 0.0}


def stored(x, dtype):
    """float64 -> (storage, its values), half saturating as the library's does."""
    if dtype == "f16":
        x = np.where(np.isnan(x), x, np.clip(x, -65504, 65504))
    b = to_bits(x, dtype)
    return b, from_bits(b, dtype)


def summed(x, residual, sum_dtype):
    """One rounding of the sum.  Two roundings, to fp32 and on to 16 bits, give the same: fp32 has twice the bits and two more."""
    return x if residual is None else stored(x + residual, sum_dtype)[1]


def normed(s, weight, eps):
    y = s / np.sqrt(np.mean(s * s, -1, keepdims=True) + eps)
    return y if weight is None else y * weight.astype(np.float64)


def gated(x, gate):
    with np.errstate(over="ignore"):
        return x if gate is None else x * gate / (1 + np.exp(-gate))


def scale_of(y):
    top = np.max(np.where(np.isnan(y), np.inf, np.abs(y)), -1)
    return np.where(np.isinf(top), np.nan, np.maximum(top / 127, TINY))


def check_codes(codes, scales, y, rel):
    """Codes and scales of float64 rows y that the kernel knows to within `rel` of each value: the scale then is off by
    rel and its own rounding, a quotient by twice that and two roundings more, times 127."""
    want = scale_of(y)
    bad = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(scales), bad)
    assert np.all(codes[bad] == 0)
    assert np.all(np.abs(scales[~bad] - want[~bad]) <= (rel + 2 * STEP32) * want[~bad])
    off = np.abs(codes[~bad].astype(np.float64) - y[~bad] / want[~bad, None])
    assert np.all(off <= 0.5 + 127 * (2 * rel + 5 * STEP32)), off.max()
    assert np.abs(codes.astype(int)).max(initial=0) <= 127


def eight(y):
    """float64 rows -> (codes int8, scales float64)."""
    s = scale_of(y)
    return np.rint(y / s[:, None]).astype(np.int8), s


def product(codes, scales, w, w_scales, bias=None, residual=None):
    """float64 result, and the magnitudes that fp32's roundings are relative to."""
    acc = codes.astype(np.float64) @ w.astype(np.float64).T             # below 2^53: exact
    p = acc * scales[:, None].astype(np.float64) * w_scales.astype(np.float64)
    out, mag = p, np.abs(p)
    for z in (bias, residual):
        if z is not None:
            out, mag = out + z, mag + np.abs(z)
    return out, mag


def logits_out(x, tokens, ranges, penalties, biases, masks):
    """x [n, V] float64; biases: a list of (ids, values) per row or None; masks: a list of bool [V] or None.  The result, and
    the magnitudes that fp32's roundings are relative to."""
    out, mag = x.copy(), np.abs(x)
    n, V = x.shape
    for i in range(n):
        if tokens is not None:
            a, b, c = (int(v) for v in ranges[i])
            a, c = max(a, 0), min(c, len(tokens))
            rep, pres, freq = (float(v) for v in penalties[i])
            ids = np.arange(a, max(a, c))
            t = tokens[a:max(a, c)].astype(np.int64)
            ok = (t >= 0) & (t < V)
            count = np.bincount(t[ok & (ids >= b)], minlength=V)
            seen = np.bincount(t[ok], minlength=V) > 0
            o = out[i]
            with np.errstate(invalid="ignore"):
                o[seen] = np.where(o[seen] > 0, o[seen] / rep, o[seen] * rep)
            mag[i] = np.abs(o) + np.abs(freq * count) + np.abs(pres)
            o[count > 0] -= freq * count[count > 0] + pres
        if biases is not None:
            last = {}
            for t, v in zip(*biases[i]):
                if 0 <= t < V:
                    last[int(t)] = float(v)
            for t, v in last.items():
                out[i, t] += v
                mag[i, t] += abs(v)
        if masks is not None and masks[i] is not None:
            out[i, ~masks[i]] = -np.inf
    return out, mag


def chosen(out):
    """The lowest token of the largest logit that is neither NaN nor -inf; -1 for none."""
    x = np.where(np.isnan(out), -np.inf, out)
    top = x.max(1)
    return np.where(top == -np.inf, -1, np.argmax(x == top[:, None], 1)).astype(np.int32)


def mask_words(allowed):
    """bool [n, V] -> uint32 [n, ceil(V / 32)]."""
    n, V = allowed.shape
    bits = np.zeros((n, -(-V // 32) * 32), bool)
    bits[:, :V] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view("<u4")
