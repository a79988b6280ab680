"""The decoder's cache operators on their own: one pass each through the package's public entry points
(`own`), or in plain torch.

  append   qk_norm_rope_append: the query and key heads of a fused projection normalised (RMS, per head),
           rotated, the keys and values written into the paged cache; then the written rows read back
           (paged_kv_read).  Pages of bf16, half or MXFP4.
  window   gqa_window_attention_paged: 1 .. 8 query positions per sequence over a sliding window and the
           first few keys (sinks), whose pages alone are still held.  Pages of bf16, half or MXFP4.
  prefill  gqa_prefill_paged: the attention of a ragged batch of new tokens over their sequences' caches,
           causal, with a window and sinks.

Head layouts are those of the framework's decode cases: 32 query / 8 kv heads of 128, 16/2 of 64, 8/8 of 64,
and 28/4 of 128 (a group of 7).  8,192 keys is the sliding window of the decoder that the framework's paged
attention serves.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
PAGE = 16                                # keys per page
BLOCK = 32                               # channels per MXFP4 block
EPS = 2.0 ** -20
THETA = 1e6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HEADS = [(32, 8, 128), (16, 2, 64), (8, 8, 64), (28, 4, 128)]


def _package():
    name = "universal_dictator_amd"
    if name not in sys.modules:
        path = os.path.join(ROOT, "universal-dictator_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location(name, path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---------------------------------------------------------------- the cases

def listed():
    wide = dict(q_heads=32, kv_heads=8, head_dim=128)
    return [
        # one dictation session: each token's heads into half pages, all in fp32 up to the cache
        dict(wide, name="append_1_f16", kind="append", n=1, rows_min=1, rows_max=1, past_max=9000, dtype="f32", pages="f16", norm=False),
        # one token for each of 64 sequences with long contexts, cache in 4 bits
        dict(wide, name="append_64_mxfp4", kind="append", n=64, rows_min=1, rows_max=1, past_max=120000, dtype="bf16", pages="mxfp4", norm=True),
        # three prompts of a small model, half precision
        dict(name="append_3x500_f16", kind="append", n=3, rows_min=307, rows_max=693, past_max=100, dtype="f16", pages="f16", norm=True, q_heads=16, kv_heads=2, head_dim=64),
        # a batch of long prompts into 4-bit pages
        dict(wide, name="append_5x1640_mxfp4", kind="append", n=5, rows_min=811, rows_max=2469, past_max=5000, dtype="bf16", pages="mxfp4", norm=True),
        # one dictation session past its window of 8,192 tokens: half pages, fp32 queries and output
        dict(wide, name="window_1_f16", kind="window", n=1, queries=1, ctx_min=30011, ctx_max=30011, window=8192, sinks=0, dtype="f32", pages="f16"),
        # a serving batch whose long sequences keep a window of 4,096 keys and 4 sinks
        dict(wide, name="window_64_bf16", kind="window", n=64, queries=1, ctx_min=500, ctx_max=20000, window=4096, sinks=4, dtype="bf16", pages="bf16"),
        # four draft tokens for each of a dozen sequences, 4-bit cache, window and sinks
        dict(wide, name="window_12x4_mxfp4", kind="window", n=12, queries=4, ctx_min=300, ctx_max=60000, window=8192, sinks=20, dtype="f32", pages="mxfp4"),
        # one session that keeps its whole long context in 4 bits
        dict(wide, name="decode_1_mxfp4", kind="window", n=1, queries=1, ctx_min=130003, ctx_max=130003, window=0, sinks=0, dtype="bf16", pages="mxfp4"),
        # a serving batch with its whole contexts in 4 bits
        dict(wide, name="decode_64_mxfp4", kind="window", n=64, queries=1, ctx_min=512, ctx_max=8192, window=0, sinks=0, dtype="bf16", pages="mxfp4"),
        # one prompt of a dictation session
        dict(wide, name="prefill_1x1131_f16", kind="prefill", n=1, rows_min=1131, rows_max=1131, past_max=0, window=8192, sinks=0, dtype="f16", pages="f16"),
        # pieces of several prompts beside their earlier pieces, which the cache holds in 4 bits
        dict(wide, name="prefill_6x300_mxfp4", kind="prefill", n=6, rows_min=37, rows_max=563, past_max=12000, window=0, sinks=0, dtype="bf16", pages="mxfp4"),
        # one long prompt of a model with a window of 4,096 and 4 sinks
        dict(wide, name="prefill_1x8192_bf16", kind="prefill", n=1, rows_min=8192, rows_max=8192, past_max=0, window=4096, sinks=4, dtype="bf16", pages="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "window", "window", "prefill"])
    hq, hkv, hd = rng.choice([HEADS[0]] + HEADS)
    c = dict(kind=kind, q_heads=hq, kv_heads=hkv, head_dim=hd)
    pages = rng.choice(["bf16", "f16", "mxfp4", "mxfp4"])
    if kind == "append":
        dtype = rng.choice(["bf16", "f16", "f32"]) if pages == "mxfp4" else rng.choice([pages, pages, "f32"])
        n = _log(rng, 1, 64)
        hi = rng.choice([1, _log(rng, 1, max(1, 8000 // n))])
        return dict(c, n=n, rows_min=max(1, hi // rng.randint(1, 4)), rows_max=hi, past_max=_log(rng, 1, 120000),
                    dtype=dtype, pages=pages, norm=rng.random() < 0.7)
    window, sinks = rng.choice([(0, 0), (_log(rng, 100, 8192), rng.choice([0, 4, rng.randint(1, 64)]))])
    if kind == "window":
        dtype = rng.choice(["bf16", "f16", "f32"]) if pages == "mxfp4" else rng.choice([pages, "f32"])
        n, queries = _log(rng, 1, 64), rng.choice([1, 1, rng.randint(2, 8)])
        held = min(window or 10**9, 480000 // n)     # keys a sequence holds
        ctx = _log(rng, 64, 100000 if window else max(65, held))
        return dict(c, n=n, queries=queries, ctx_min=max(8, ctx // rng.randint(1, 8)), ctx_max=ctx,
                    window=held if window else 0, sinks=sinks, dtype=dtype, pages=pages)
    dtype = rng.choice(["bf16", "f16"]) if pages == "mxfp4" else pages
    n = _log(rng, 1, 8)
    hi = _log(rng, 9, 5000 // n)
    past = rng.choice([0, min(24000, _log(rng, 20, 16 * 10**6 // (n * hi)))])
    return dict(c, n=n, rows_min=max(1, hi // rng.randint(1, 6)), rows_max=hi, past_max=past, window=window,
                sinks=sinks, dtype=dtype, pages=pages)


# ---------------------------------------------------------------- helpers

class Buf:
    """Device memory of a torch tensor, as the package takes it."""

    def __init__(self, t):
        self.ptr, self.nbytes = t.data_ptr(), t.numel() * t.element_size()


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + 17) % (1 << 60))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _spread(lo, hi, n):
    """n sizes from lo to hi, evenly apart."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _inv_freq(hd):
    i = torch.arange(hd // 2, dtype=torch.float64, device=DEV)
    return (THETA ** (-2.0 * i / hd)).float()


def _shuffled(v, seed):
    g = torch.Generator()
    g.manual_seed(int(seed) * 31 + 7)
    return [v[i] for i in torch.randperm(len(v), generator=g).tolist()]


def _lens(case, seed):
    """(new tokens, tokens before them) of each sequence."""
    n = case["n"]
    if case["kind"] == "window":
        ctx = _shuffled(_spread(case["ctx_min"], case["ctx_max"], n), seed)
        new = [min(case["queries"], c) for c in ctx]
        return new, [c - m for c, m in zip(ctx, new)]
    new = _shuffled(_spread(case["rows_min"], case["rows_max"], n), seed)
    return new, _shuffled(_spread(case["past_max"] // 3, case["past_max"], n), seed + 1)


def _held(case, new, past):
    """The first key of the window and the first behind the sinks for a sequence's first new token."""
    lo = max(0, past + 1 - case["window"]) if case["window"] else 0
    return lo, min(case["sinks"], lo)


def _pages(case, new, past, g):
    """The page table (-1 where a page has been given back) and the pools' number of pages."""
    n = len(new)
    most = max(-(-(p + t) // PAGE) for p, t in zip(past, new))
    held = []
    for p, t in zip(past, new):
        if case["kind"] == "append":
            first, sink = p, 0
        else:
            first, sink = _held(case, t, p)
        held.append(sorted(set(range(-(-sink // PAGE))) | set(range(first // PAGE, -(-(p + t) // PAGE)))))
    total = sum(len(h) for h in held)
    order = torch.randperm(total + 5, generator=g, device=DEV).int()
    table = torch.full((n, most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, h in enumerate(held):
        table[i, torch.tensor(h, device=DEV)] = order[at:at + len(h)]
        at += len(h)
    return table, total + 5


def _block_exponent(amax):
    """The smallest power of two that brings a block's largest magnitude to 7 or less, as an exponent."""
    f, x = torch.frexp(amax)
    return torch.where(amax == 0, torch.full_like(x, -100), torch.where(f <= 0.875, x - 3, x - 2).clamp(min=-100))


def _fp4_rows(x):
    """Rows [.., D] as MXFP4 holds them: (levels' values, exponents), each value to the nearest of 0, 0.5, 1,
    1.5, 2, 3, 4, 6 times the block's power of two, ties to the even code."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    e = _block_exponent(b.abs().amax(-1, keepdim=True))
    y = torch.ldexp(b.abs(), -e)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    return (torch.round(y / step) * step).clamp(max=6) * torch.sign(b), e


def _fp4_pages(g, total, hkv, hd, scale):
    """A pool of MXFP4 pages of normal keys or values: [pages, kv heads, 16 hd / 2 + 16 hd / 32] bytes, the
    rows' codes (low nibble first), then the rows' exponents + 127."""
    pool = torch.empty(total, hkv, PAGE * hd // 2 + PAGE * hd // BLOCK, dtype=torch.uint8, device=DEV)
    for a in range(0, total, 4096):
        x = _randn(g, min(4096, total - a), hkv, PAGE, hd) * scale
        v, e = _fp4_rows(x)
        m = (2 * v.abs()).flatten(-2).int()               # 0, 1, 2, 3, 4, 6, 8, 12
        code = torch.where(m <= 4, m, torch.where(m == 6, 5, torch.where(m == 8, 6, 7))) + 8 * (v.flatten(-2) < 0).int()
        pool[a:a + 4096, :, :PAGE * hd // 2] = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8).flatten(-2)
        pool[a:a + 4096, :, PAGE * hd // 2:] = (e.squeeze(-1) + 127).to(torch.uint8).flatten(-2)
    return pool


def prepare(case, seed):
    g = _gen(seed)
    hq, hkv, hd, n = case["q_heads"], case["kv_heads"], case["head_dim"], case["n"]
    new, past = _lens(case, seed)
    table, total = _pages(case, new, past, g)
    rows, t = sum(new), TYPES[case["dtype"]]
    dev = dict(dtype=torch.int32, device=DEV)
    s = dict(case, table=table, total=total, rows=rows, most=table.shape[1])
    # a few channels of a key head are larger than the rest
    channel = torch.exp(0.5 * _randn(g, hkv, 1, hd))
    if case["kind"] == "append":
        qkv = _randn(g, rows, (hq + 2 * hkv) * hd).to(t)                # the fused projection's rows
        shape = (total, hkv, PAGE, hd) if case["pages"] != "mxfp4" else (total, hkv, PAGE * hd // 2 + PAGE * hd // BLOCK)
        kind = TYPES.get(case["pages"], torch.uint8)
        s.update(qkv=qkv, q_out=torch.empty(rows, hq * hd, dtype=t, device=DEV), inv_freq=_inv_freq(hd),
                 kp=torch.zeros(shape, dtype=kind, device=DEV), vp=torch.zeros(shape, dtype=kind, device=DEV),
                 pos=torch.tensor([p + i for p, m in zip(past, new) for i in range(m)], **dev),
                 seqs=torch.tensor([i for i, m in enumerate(new) for _ in range(m)], **dev),
                 qw=(1 + 0.2 * _randn(g, hd)) if case["norm"] else None, kw=torch.exp(0.5 * _randn(g, hd)) if case["norm"] else None)
        back = torch.float32 if case["pages"] == "mxfp4" else kind
        s.update(k_back=torch.empty(rows, hkv * hd, dtype=back, device=DEV), v_back=torch.empty(rows, hkv * hd, dtype=back, device=DEV))
        return s
    if case["pages"] == "mxfp4":
        s.update(kp=_fp4_pages(g, total, hkv, hd, channel), vp=_fp4_pages(g, total, hkv, hd, 1.0))
    else:
        kind = TYPES[case["pages"]]
        s.update(kp=(_randn(g, total, hkv, PAGE, hd) * channel).to(kind), vp=_randn(g, total, hkv, PAGE, hd).to(kind))
    ends = [[p + i + 1 for i in range(m)] for p, m in zip(past, new)]
    if case["kind"] == "window":
        M = case["queries"]
        ends = [[0] * (M - len(e)) + e for e in ends]                   # a short sequence's missing rows are empty
    first = [[max(0, e - case["window"]) if case["window"] else 0 for e in v] for v in ends]
    flat = torch.tensor([[a, e] for f, v in zip(first, ends) for a, e in zip(f, v)], **dev)
    nq = flat.shape[0]
    s.update(q=_randn(g, nq, hq * hd).to(t), ranges=flat, out=torch.empty(nq, hq * hd, dtype=t, device=DEV),
             span=max(p + m - _held(case, m, p)[0] for p, m in zip(past, new)), most_rows=max(new), rows=nq)
    if case["kind"] == "prefill":
        s["q_start"] = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), **dev)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "append":
        return _plain_append(s)
    return _plain_window(s) if s["kind"] == "window" else _plain_prefill(s)


def _run_own(s):
    ud = _package()
    hq, hkv, hd = s["q_heads"], s["kv_heads"], s["head_dim"]
    kp, vp, table = Buf(s["kp"]), Buf(s["vp"]), Buf(s["table"])
    if s["kind"] == "append":
        qkv = s["qkv"]
        ld = qkv.shape[1]
        q, k, v = Buf(qkv), Buf(qkv[:, hq * hd:]), Buf(qkv[:, (hq + hkv) * hd:])
        pos, seqs, kb, vb = Buf(s["pos"]), Buf(s["seqs"]), Buf(s["k_back"]), Buf(s["v_back"])
        ud.qk_norm_rope_append(q, k, v, Buf(s["q_out"]), kp, vp, s["total"], table, s["n"], s["most"], pos, s["rows"], hq, hkv, hd,
                               seqs=seqs, q_weight=Buf(s["qw"]) if s["norm"] else None, k_weight=Buf(s["kw"]) if s["norm"] else None,
                               eps=EPS, inv_freq=Buf(s["inv_freq"]), dtype=s["dtype"], kv_format=s["pages"], q_ld=ld, k_ld=ld, v_ld=ld)
        ud.paged_kv_read(kp, vp, s["total"], table, s["n"], s["most"], pos, kb, vb, s["rows"], hkv, hd, seqs=seqs,
                         dtype="f32" if s["pages"] == "mxfp4" else s["pages"], kv_format=s["pages"])
        return s["q_out"], s["k_back"], s["v_back"]
    if s["kind"] == "window":
        if "ws" not in s:
            s["ws"] = torch.empty(ud.gqa_window_workspace_bytes(s["n"], s["queries"], hq, hkv, hd, s["sinks"], s["span"]) + 16, dtype=torch.uint8, device=DEV)
        ud.gqa_window_attention_paged(Buf(s["q"]), kp, vp, s["total"], table, s["most"], Buf(s["ranges"]), s["sinks"], Buf(s["out"]), s["n"],
                                      s["queries"], hq, hkv, hd, s["span"], Buf(s["ws"]), dtype=s["dtype"], kv_format=s["pages"])
        return s["out"]
    if "ws" not in s:
        s["ws"] = torch.empty(ud.gqa_prefill_workspace_bytes(s["n"], s["rows"], s["most_rows"], hq, hkv, hd, s["sinks"], s["span"]) + 16, dtype=torch.uint8, device=DEV)
    ud.gqa_prefill_paged(Buf(s["q"]), kp, vp, s["total"], table, s["most"], Buf(s["q_start"]), Buf(s["ranges"]), s["sinks"], Buf(s["out"]), s["n"],
                         s["rows"], s["most_rows"], hq, hkv, hd, s["span"], Buf(s["ws"]), dtype=s["dtype"], kv_format=s["pages"])
    return s["out"]


def _turned(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _plain_append(s):
    hq, hkv, hd, rows = s["q_heads"], s["kv_heads"], s["head_dim"], s["rows"]
    q, k, v = s["qkv"].split([hq * hd, hkv * hd, hkv * hd], -1)
    angle = s["pos"].double()[:, None, None] * s["inv_freq"].double()   # far positions: fp32 angles would be off by 1e-2
    cos, sin = angle.cos(), angle.sin()
    q = _turned(_normed(q.float().view(rows, hq, hd), s["qw"]), cos.float(), sin.float())
    if s["pages"] == "mxfp4":                                           # values next to a border between two codes: 64 bits
        k = _turned(_normed(k.double().view(rows, hkv, hd), s["kw"]), cos, sin)
        k, v = (torch.ldexp(*_fp4_rows(x)).float() for x in (k, v.view(rows, hkv, hd)))
    else:
        k = _turned(_normed(k.float().view(rows, hkv, hd), s["kw"]), cos.float(), sin.float()).to(s["k_back"].dtype)
        v = v.to(s["v_back"].dtype)
    return q.reshape(rows, -1).to(s["qkv"].dtype), k.reshape(rows, -1), v.reshape(rows, -1)


def _dense(s, pool, blocks):
    """The keys or values of page-table blocks [n, B] (-1: none) as fp32 [n, kv heads, 16 B, D]."""
    hkv, hd = s["kv_heads"], s["head_dim"]
    page = torch.gather(s["table"], 1, blocks.clamp(min=0)).clamp(min=0).long()
    x = pool[page]
    if s["pages"] == "mxfp4":
        c = x[..., :PAGE * hd // 2].unflatten(-1, (PAGE, hd // 2))
        c = torch.stack([c & 15, c >> 4], -1).flatten(-2).int()
        e = x[..., PAGE * hd // 2:].unflatten(-1, (PAGE, hd // BLOCK)).int() - 127
        levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=DEV)
        x = torch.ldexp(levels[c].unflatten(-1, (-1, BLOCK)), e.unsqueeze(-1)).flatten(-2)
    return x.float().transpose(1, 2).reshape(len(blocks), hkv, -1, hd)


def _attend(s, q, ranges):
    """q [n, T, Hq, D], ranges [n, T, 2] over sinks and the span of each sequence's ranges -> [n, T, Hq, D]."""
    n, T, hq, hd = q.shape
    hkv, sinks = s["kv_heads"], s["sinks"]
    lo, hi = ranges[..., 0], ranges[..., 1]
    some = lo < hi
    first = torch.where(some, lo, 1 << 30).amin(1) // PAGE
    wide = (s["span"] + PAGE - 2) // PAGE + 1
    sunk = -(-sinks // PAGE)
    blocks = torch.cat([torch.arange(sunk, device=DEV).expand(n, -1), first[:, None] + torch.arange(wide, device=DEV)], 1)
    twice = torch.cat([blocks[:, :sunk] >= first[:, None], blocks[:, sunk:] >= s["table"].shape[1]], 1)
    blocks = torch.where(twice, -1, blocks)
    j = torch.where(blocks[..., None] < 0, 1 << 30, blocks[..., None] * PAGE + torch.arange(PAGE, device=DEV)).flatten(1)[:, None, :]
    lo, hi = lo[..., None], hi[..., None]
    seen = ((j >= lo) & (j < hi) | (j < sinks) & (j < lo)) & some[..., None]            # [n, T, keys]
    k, v = _dense(s, s["kp"], blocks.long()), _dense(s, s["vp"], blocks.long())
    v = torch.where(seen.any(1)[:, None, :, None], v, 0)
    qq = q.float().view(n, T, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, hd) * (hd ** -0.5)
    p = torch.matmul(qq, k.transpose(2, 3).contiguous()).view(n, hkv, hq // hkv, T, -1)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m == -math.inf, 0, m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, p.shape[-1]), v).view(n, hkv, hq // hkv, T, hd)
    o = torch.where(total > 0, o / total, 0)
    return o.permute(0, 3, 1, 2, 4).reshape(n, T, hq, hd)


def _plain_window(s):
    n, M = s["n"], s["queries"]
    return _attend(s, s["q"].view(n, M, s["q_heads"], -1), s["ranges"].view(n, M, 2)).reshape(n * M, -1).to(s["q"].dtype)


def _plain_prefill(s):
    n, T, rows = s["n"], s["most_rows"], s["rows"]
    start = s["q_start"].long()
    at = start[:-1, None] + torch.arange(T, device=DEV)
    real = at < start[1:, None]
    at = torch.where(real, at, 0)
    ranges = torch.where(real[..., None], s["ranges"][at], 0)
    o = _attend(s, s["q"].view(rows, s["q_heads"], -1)[at], ranges).to(s["q"].dtype)
    row = torch.arange(rows, device=DEV)
    seq = torch.bucketize(row, start[1:], right=True)
    return o[seq, row - start[seq]].reshape(rows, -1)


# ---------------------------------------------------------------- work

def _row_bytes(case):
    """Bytes of a key's row of one kv head."""
    hd = case["head_dim"]
    return hd // 2 + hd // BLOCK if case["pages"] == "mxfp4" else 2 * hd


def work(case):
    hq, hkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    size = 4 if case["dtype"] == "f32" else 2
    new, past = _lens(case, 0)
    if case["kind"] == "append":
        rows, back = sum(new), 4 if case["pages"] == "mxfp4" else 2
        # the fused rows in, q out, the cache rows in and out of the pages, and the rows read back
        each = (2 * hq + 2 * hkv) * hd * size + 2 * hkv * (2 * _row_bytes(case) + back * hd)
        return {"bytes": rows * each, "flops": rows * (hq + hkv) * hd * 7}
    pairs = keys = 0
    W = case["window"] or 1 << 40
    for t, p in zip(new, past):
        lo, sunk = _held(case, t, p)
        keys += p + t - lo + sunk
        full = max(0, min(t, p + t - W))                     # rows whose window is full: their ends are past W
        pairs += full * W + sum(range(p + 1, p + t - full + 1)) + sum(min(case["sinks"], max(0, e - W)) for e in range(p + 1, p + t + 1)) \
            if case["window"] else sum(range(p + 1, p + t + 1))
    rows = case["n"] * case["queries"] if case["kind"] == "window" else sum(new)
    return {"bytes": 2 * rows * hq * hd * size + 2 * keys * hkv * _row_bytes(case), "flops": pairs * hq * hd * 4}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["kind"] == "append" else _exact_attention(s)


def _exact_fp4(x):
    """MXFP4's values of float64 rows, by the borders between the levels."""
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2
    for _ in range(2):                                       # the logarithm may be off by one at a power of two
        e = torch.where(top > 7 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 7 * torch.exp2(e - 1), e - 1, e)
    unit = torch.exp2(e)
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    mid = (levels[1:] + levels[:-1]) / 2
    y = b.abs() / unit
    below, above = torch.bucketize(y, mid, right=False), torch.bucketize(y, mid, right=True)
    code = torch.where(below % 2 == 0, below, above)         # on a border: the even one of the two codes
    return (levels[code] * unit * torch.sign(b)).reshape(x.shape)


def _exact_append(s):
    hq, hkv, hd, rows = s["q_heads"], s["kv_heads"], s["head_dim"], s["rows"]
    x = s["qkv"].double().view(rows, hq + 2 * hkv, hd)
    w = s["pos"].double()[:, None] * s["inv_freq"].double()[None]
    turn = torch.polar(torch.ones_like(w), w)[:, None]

    def heads(y, weight):
        if weight is not None:
            y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=-1, keepdim=True) ** 2 / hd + EPS) * weight.double()
        z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = heads(x[:, :hq], s["qw"]), heads(x[:, hq:hq + hkv], s["kw"]), x[:, hq + hkv:]
    if s["pages"] == "mxfp4":
        k, v = _exact_fp4(k), _exact_fp4(v)
    return q.reshape(rows, -1), k.reshape(rows, -1), v.reshape(rows, -1)


def _exact_rows(s, pool, i, keys):
    """Keys (a list of positions) of sequence i as float64 [kv heads, keys, D]."""
    hd = s["head_dim"]
    x = pool[s["table"][i][keys // PAGE].long(), :, :]
    r = keys % PAGE
    if s["pages"] != "mxfp4":
        return x[torch.arange(len(keys), device=DEV), :, r].transpose(0, 1).double()
    code = x[:, :, :PAGE * hd // 2].reshape(len(keys), -1, PAGE, hd // 2)[torch.arange(len(keys), device=DEV), :, r].int()
    scale = x[:, :, PAGE * hd // 2:].reshape(len(keys), -1, PAGE, hd // BLOCK)[torch.arange(len(keys), device=DEV), :, r]
    c = torch.empty(*code.shape[:-1], hd, dtype=torch.int32, device=DEV)
    c[..., 0::2], c[..., 1::2] = code % 16, code // 16
    m, exp = c % 2, c // 2 % 4                               # e2m1: sign, two exponent bits, one mantissa bit
    mag = torch.where(exp == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(exp.double() - 1))
    return (torch.where(c >= 8, -mag, mag) * torch.exp2(scale.double() - 127).repeat_interleave(BLOCK, -1)).transpose(0, 1)


def _exact_attention(s):
    n, hq, hkv, hd = s["n"], s["q_heads"], s["kv_heads"], s["head_dim"]
    start = s["q_start"].tolist() if s["kind"] == "prefill" else [i * s["queries"] for i in range(n + 1)]
    ranges = s["ranges"].tolist()
    out = torch.zeros(len(ranges), hq, hd, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(-1, hq, hd)
    for i in range(n):
        at = [r for r in range(start[i], start[i + 1]) if ranges[r][0] < ranges[r][1]]
        for a in range(0, len(at), 1024):
            some = at[a:a + 1024]
            lo, hi = min(ranges[r][0] for r in some), max(ranges[r][1] for r in some)
            keys = torch.tensor(list(range(min(s["sinks"], lo))) + list(range(lo, hi)), device=DEV)
            k, v = _exact_rows(s, s["kp"], i, keys), _exact_rows(s, s["vp"], i, keys)
            lim = torch.tensor([ranges[r] for r in some], device=DEV)
            hide = ~((keys < lim[:, 1:]) & ((keys >= lim[:, :1]) | (keys < s["sinks"])))
            for h in range(hq):
                z = q[some, h] @ k[h // (hq // hkv)].T / math.sqrt(hd)
                out[some, h] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v[h // (hq // hkv)]
    return out.view(len(ranges), -1)
