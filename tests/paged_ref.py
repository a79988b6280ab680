"""Plain float64 forms of the paged-cache operators (include/ud_decode.h): page formats, the fused norm / rotation /
append, windowed attention with sinks.  numpy only; used by the tests of those calls."""
import numpy as np

PAGE, BLOCK = 16, 32
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
# A rounding's half step relative to the value: with p significant bits a value in [2^e, 2^(e+1)) is off by at most
# 2^(e-p), which is 2^-p of the value at the binade's start.  p = 8, 11, 24.
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def to_bits(x, dtype):
    """float array -> storage of dtype (uint16 for 16-bit types, float32)."""
    if dtype == "bf16":
        return bf16_bits(np.asarray(x, np.float32))
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return np.asarray(x, np.float32).astype(np.float16).view(np.uint16)
    return np.asarray(x, np.float32)


def from_bits(b, dtype):
    """storage of dtype -> float64."""
    if dtype == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return b.astype(np.float64)


def rounded(x, dtype):
    return from_bits(to_bits(x, dtype), dtype)


# ---------------------------------------------------------------- MXFP4

def fp4_encode(x):
    """x [.., D] float64 -> (codes uint8 [.., D], exponent bytes uint8 [.., D / 32])."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, BLOCK)
    mag = np.abs(b)
    top = np.max(np.where(np.isnan(mag), np.inf, mag), -1)
    bad = ~np.isfinite(top)
    safe = np.where(bad | (top == 0), 1.0, top)
    f, e2 = np.frexp(safe)                       # top = f 2^e2, 0.5 <= f < 1;  <= 7 2^E  <=>  f <= 7/8 2^(E + 3 - e2)
    e = np.where(f <= 0.875, e2 - 3, e2 - 2)
    e = np.where(top == 0, -100, np.clip(e, -100, 125))
    with np.errstate(invalid="ignore"):
        y = np.where(bad[..., None], 0.0, mag) / np.exp2(e.astype(np.float64))[..., None]
    code = np.zeros(y.shape, np.uint8)
    for k, (lo, hi) in enumerate(zip(LEVELS[:-1], LEVELS[1:])):
        mid = (lo + hi) / 2
        code += ((y > mid) | ((y == mid) & (k % 2 == 1))).astype(np.uint8)      # a tie goes to the even code
    code |= (np.signbit(b).astype(np.uint8) << 3)
    return code.reshape(x.shape), np.where(bad, 255, e + 127).astype(np.uint8)


def fp4_decode(code, byte):
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    return (v.reshape(*code.shape[:-1], -1, BLOCK) * s[..., None]).reshape(code.shape)


def held(x, fmt):
    """The values that pages of fmt hold for rows x [.., D]."""
    return fp4_decode(*fp4_encode(x)) if fmt == "mxfp4" else rounded(x, fmt)


# ---------------------------------------------------------------- pages

def page_bytes(fmt, d):
    return PAGE * (d // 2 + d // BLOCK) if fmt == "mxfp4" else PAGE * 2 * d


def new_pool(fmt, num_blocks, hkv, d):
    """Pages of NaN: what is not written must not be seen."""
    return np.full((num_blocks, hkv, page_bytes(fmt, d)), 0xFF, np.uint8)


def put_row(pool, fmt, d, page, row, x):
    """Row `row` of a page from x [hkv, d] float64 (values that the format holds)."""
    if fmt == "mxfp4":
        code, byte = fp4_encode(x)
        pool[page, :, row * d // 2:(row + 1) * d // 2] = code[:, 0::2] | code[:, 1::2] << 4
        at = PAGE * d // 2 + row * (d // BLOCK)
        pool[page, :, at:at + d // BLOCK] = byte
    else:
        pool[page, :, row * 2 * d:(row + 1) * 2 * d] = to_bits(x, fmt).view(np.uint8).reshape(len(x), 2 * d)


def get_row(pool, fmt, d, page, row):
    if fmt == "mxfp4":
        c = pool[page, :, row * d // 2:(row + 1) * d // 2]
        code = np.stack([c & 15, c >> 4], -1).reshape(len(c), d)
        at = PAGE * d // 2 + row * (d // BLOCK)
        return fp4_decode(code, pool[page, :, at:at + d // BLOCK])
    b = np.ascontiguousarray(pool[page, :, row * 2 * d:(row + 1) * 2 * d])
    return from_bits(b.view(np.uint16), fmt)


def assign_pages(rng, lens, spare=3, keep=None):
    """Block tables for sequences of lens keys: random distinct pages; entries without a page hold junk outside the pool.
    keep(i, block) -> bool: whether the sequence still holds the page."""
    n, most = len(lens), max(1, max(-(-L // PAGE) for L in lens))
    want = [(i, b) for i, L in enumerate(lens) for b in range(-(-L // PAGE)) if keep is None or keep(i, b)]
    num = len(want) + spare
    pages = rng.permutation(num)[:len(want)]
    table = np.where(rng.random((n, most)) < 0.5, -1 - rng.integers(0, 2 ** 30, (n, most)), num + rng.integers(0, 2 ** 30, (n, most))).astype(np.int32)
    for (i, b), p in zip(want, pages):
        table[i, b] = p
    return table, num


def fill(pool, table, fmt, d, seqs, num):
    """seqs: per sequence [L, hkv, d] float64 values; rows of pages that are not held are left out."""
    for i, s in enumerate(seqs):
        for j in range(len(s)):
            p = table[i, j // PAGE]
            if 0 <= p < num:
                put_row(pool, fmt, d, p, j % PAGE, s[j])


# ---------------------------------------------------------------- the operators

def norm_rope(x, weight, eps, pos, inv_freq):
    """x [rows, heads, d] float64."""
    y = np.asarray(x, np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * weight.astype(np.float64)
    if inv_freq is not None:
        a = pos.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
        h = y.shape[-1] // 2
        u, v = y[..., :h], y[..., h:]
        y = np.concatenate([u * np.cos(a) - v * np.sin(a), v * np.cos(a) + u * np.sin(a)], -1)
    return y


def visible(lo, hi, sinks, limit):
    """Keys that a range sees."""
    lo, hi = max(lo, 0), min(hi, limit)
    if lo >= hi:
        return np.zeros(0, np.int64)
    return np.concatenate([np.arange(min(sinks, lo)), np.arange(lo, hi)])


def attend(q, k, v, keys, scale):
    """One query row of one head: q [d], k, v [L, d] -> (out, sum p |v|, max |score|, max sum |q||k| scale)."""
    if not len(keys):
        return np.zeros(v.shape[1]), np.zeros(v.shape[1]), 0.0, 0.0
    kk, vv = k[keys], v[keys]
    s = kk @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ vv, p @ np.abs(vv), np.abs(s).max(), (np.abs(kk) @ np.abs(q)).max() * scale


def attention(q, kseqs, vseqs, seq_of, ranges, sinks, hkv, limit, held_keys=None):
    """q [rows, hq, d] float64, kseqs / vseqs per sequence [L, hkv, d]; returns (out, |v|-weighted, bounds of the scores).
    held_keys(i) -> bool [L]: keys whose pages the sequence holds."""
    rows, hq, d = q.shape
    out, mag = np.zeros_like(q), np.zeros_like(q)
    top, dot = np.zeros((rows, hq)), np.zeros((rows, hq))
    count = np.zeros(rows)
    for r in range(rows):
        i = seq_of[r]
        keys = visible(int(ranges[r, 0]), int(ranges[r, 1]), sinks, limit)
        if held_keys is not None:
            keys = keys[held_keys(i)[keys]]
        count[r] = len(keys)
        for h in range(hq):
            g = h // (hq // hkv)
            out[r, h], mag[r, h], top[r, h], dot[r, h] = attend(q[r, h], kseqs[i][:, g], vseqs[i][:, g], keys, d ** -0.5)
    return out, mag, top, dot, count


def attention_tolerance(ref, mag, top, dot, count, d, dtype, p_step):
    """Elementwise: the scores' fp32 sums (d + 8 roundings of at most sum |q||k|), the exponent's argument (4 roundings of
    the largest score in binary digits), the sums over the keys (a lane adds every 16th, the products every 32nd), each
    probability's own rounding p_step, the result's rounding."""
    gamma = 2.0 ** -24 * (2 * (d + 8) * dot + 4 * 1.4427 * top + (count / 16 + 64)[:, None])
    return (gamma[..., None] + p_step) * mag * 1.02 + HALF_STEP[dtype] * np.abs(ref) * 1.01 + 1e-30
