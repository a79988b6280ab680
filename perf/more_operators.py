"""What a decoder does between two attentions and after the last one, in 8 bits: one pass each through the package's
public entry points (`own`), or in plain torch.

  norm     rms_norm: the residual's addition and the root-mean-square norm, out in the rows' type.
  linear   rms_norm with its output in 8 bits (a scale per token), then i8_linear: a layer's way into attention or
           into its gate and up projections.
  product  i8_linear alone: int8 rows times int8 weights, scales for each token and each channel.
  down     i8_quantize with the gate (silu(gate) * up in 8 bits), then i8_linear with the residual added.
  logits   logits_process: penalties for repeated tokens, biases, grammar masks, and the greedy token.

Widths: 4,096 -> 6,144 is the fused q, k and v of the framework's decode cases (32 + 8 + 8 heads of 128), 1,024 the
encoder's width (4,096 its feed-forward one), 1,025 the RNN-T vocabulary; the others are generic.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
EPS = 2.0 ** -20
TINY = 2.0 ** -126
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


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
    return [
        # one dictation session: the norm in front of the head, one token
        dict(name="norm_1_bf16", kind="norm", rows=1, dim=4096, dtype="bf16", sums="bf16", residual=True),
        # a batch of prompts at the encoder's width, the residual kept in fp32
        dict(name="norm_8200_f16", kind="norm", rows=8200, dim=1024, dtype="f16", sums="f32", residual=True),
        # one token into the fused q, k and v
        dict(name="linear_1_bf16", kind="linear", rows=1, dim=4096, out=6144, dtype="bf16", sums="bf16", residual=True, bias=False),
        # a serving batch of 64 tokens
        dict(name="linear_64_bf16", kind="linear", rows=64, dim=4096, out=6144, dtype="bf16", sums="f32", residual=True, bias=True),
        # a piece of a prompt
        dict(name="linear_563_f16", kind="linear", rows=563, dim=4096, out=6144, dtype="f16", sums="f16", residual=True, bias=False),
        # a batch of long prompts
        dict(name="linear_8192_bf16", kind="linear", rows=8192, dim=4096, out=6144, dtype="bf16", sums="bf16", residual=True, bias=False),
        # the head of a small model for a dozen sequences: fp32 logits over a vocabulary of odd size
        dict(name="product_13_f32", kind="product", rows=13, dim=2048, out=32001, dtype="f32", bias=False),
        # one token through the second half of a feed-forward block
        dict(name="down_1_bf16", kind="down", rows=1, dim=12288, out=4096, dtype="bf16"),
        # a prompt of ordinary length through it
        dict(name="down_2469_bf16", kind="down", rows=2469, dim=12288, out=4096, dtype="bf16"),
        # one dictation session under a grammar, with its words' biases
        dict(name="logits_1_f32", kind="logits", rows=1, vocab=131072, dtype="f32", past=9000, new=300, biases=200, masks="all"),
        # a serving batch, some of its sequences under a grammar
        dict(name="logits_64_bf16", kind="logits", rows=64, vocab=131072, dtype="bf16", past=20000, new=2000, biases=50, masks="some"),
        # a dozen streams with a vocabulary of odd size, no grammar
        dict(name="logits_12_f16", kind="logits", rows=12, vocab=32001, dtype="f16", past=500, new=100, biases=0, masks="none"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "linear", "linear", "product", "down", "logits", "logits"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "logits":
        vocab = rng.choice([_log(rng, 1025, 131072), 131072])
        rows = _log(rng, 1, min(256, 64 * 131072 // vocab))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "f16"]), past=_log(rng, 10, 20000),
                    new=_log(rng, 1, 2000), biases=rng.choice([0, _log(rng, 1, 1000)]), masks=rng.choice(["none", "some", "all"]))
    if kind == "norm":
        dim = 8 * _log(rng, 64, 1024)
        dtype = rng.choice(["bf16", "f16", "f32"])
        return dict(kind=kind, rows=_log(rng, 1, min(16384, 8200 * 1024 // dim)), dim=dim, dtype=dtype, sums=rng.choice([dtype, "f32"]),
                    residual=rng.random() < 0.8)
    dim, out = 16 * _log(rng, 32, 768), _log(rng, 256, 16384)
    rows = _log(rng, 1, min(8192, 8192 * 4096 * 6144 // (dim * out)))
    if kind == "linear":
        return dict(kind=kind, rows=rows, dim=dim, out=out, dtype=dtype, sums=rng.choice([dtype, "f32"]), residual=rng.random() < 0.8,
                    bias=rng.random() < 0.5)
    if kind == "product":
        return dict(kind=kind, rows=rows, dim=dim, out=out, dtype=rng.choice(["f32", "bf16", "f16"]), bias=rng.random() < 0.5)
    return dict(kind=kind, rows=rows, dim=dim, out=out, dtype=dtype)


# ---------------------------------------------------------------- inputs

class Buf:
    """Device memory of a torch tensor, as the package takes it."""

    def __init__(self, t):
        self.ptr, self.nbytes = t.data_ptr(), t.numel() * t.element_size()


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + 29) % (1 << 60))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _weights(g, out, dim):
    """int8 weights [out, dim] with a scale per channel, of normal ones."""
    codes, scales = torch.empty(out, dim, dtype=torch.int8, device=DEV), torch.empty(out, device=DEV)
    for a in range(0, out, 8192):
        w = _randn(g, min(8192, out - a), dim) * dim ** -0.5
        scales[a:a + 8192] = w.abs().amax(1) / 127
        codes[a:a + 8192] = torch.round(w / scales[a:a + 8192, None]).to(torch.int8)
    return codes, scales


def _spread(lo, hi, n):
    """n sizes from lo to hi, evenly apart."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def prepare(case, seed):
    g = _gen(seed)
    s, rows, t = dict(case), case["rows"], TYPES[case["dtype"]]
    if case["kind"] == "logits":
        _prepare_logits(s, g)
    else:
        dim, out = case["dim"], case.get("out")
        channel = torch.exp(0.5 * _randn(g, dim))                      # a few channels are larger than the rest
        if case["kind"] in ("norm", "linear"):
            s["x"] = (_randn(g, rows, dim) * channel).to(t)
            s["weight"] = 1 + 0.2 * _randn(g, dim)
            if case["residual"]:
                s["res"] = (4 * _randn(g, rows, dim)).to(TYPES[case["sums"]])
                s["sum"] = torch.empty_like(s["res"])
        if case["kind"] == "norm":
            s["out_rows"] = torch.empty(rows, dim, dtype=t, device=DEV)
        else:
            s["w"], s["w_scales"] = _weights(g, out, dim)
            s["codes"] = torch.empty(rows, dim, dtype=torch.int8, device=DEV)
            s["scales"] = torch.empty(rows, device=DEV)
            s["bias_row"] = 0.3 * _randn(g, out) if case.get("bias") else None
            s["out_rows"] = torch.empty(rows, out, dtype=t, device=DEV)
        if case["kind"] == "product":
            x = _randn(g, rows, dim) * channel
            s["scales"] = x.abs().amax(1) / 127
            s["codes"] = torch.round(x / s["scales"][:, None]).to(torch.int8)
        if case["kind"] == "down":
            s["fused"] = (_randn(g, rows, 2 * dim) * torch.cat([channel, channel])).to(t)   # gate | up
            s["res"] = (4 * _randn(g, rows, out)).to(t)
    if case["kind"] == "down":
        s["up"] = s["fused"][:, case["dim"]:]
    s["buf"] = {k: Buf(v) if torch.is_tensor(v) else None for k, v in s.items()}
    return s


def _prepare_logits(s, g):
    rows, vocab = s["rows"], s["vocab"]
    i32 = dict(dtype=torch.int32, device=DEV)
    s["logits"] = (3 * _randn(g, rows, vocab)).to(TYPES[s["dtype"]])
    # each row's history: its prompt and what it has generated, frequent tokens often
    past, new = _spread(s["past"] // 3, s["past"], rows), _spread(s["new"] // 4, s["new"], rows)
    at, ranges = 0, []
    for p, m in zip(past, new):
        ranges.append([at, at + p, at + p + m])
        at += p + m
    s["tokens"] = (vocab * torch.rand(at, generator=g, device=DEV) ** 3).int().clamp_(max=vocab - 1)
    s["ranges"], s["n_tokens"] = torch.tensor(ranges, **i32), at
    # repetition, presence, frequency; every fourth row without any
    pen = torch.tensor([1.0, 0.0, 0.0], device=DEV) + torch.rand(rows, 3, generator=g, device=DEV) * torch.tensor([0.3, 0.6, 0.4], device=DEV)
    if rows > 1:
        pen[3::4] = torch.tensor([1.0, 0.0, 0.0], device=DEV)
    s["penalties"] = pen
    k = s["biases"]
    s["bias_ids"] = s["bias_values"] = s["bias_ranges"] = s["mask"] = s["mask_rows"] = None
    if k:
        ids = torch.argsort(torch.rand(rows, vocab, generator=g, device=DEV), 1)[:, :k] if rows * vocab <= 1 << 24 else \
            (torch.arange(k, device=DEV) * (vocab // k) + torch.randint(0, vocab // k, (rows, k), generator=g, device=DEV))
        s["k"] = k = ids.shape[1]
        s["bias_ids"], s["bias_values"] = ids.int().flatten(), 2 * _randn(g, rows * k) + 1
        s["bias_ranges"] = torch.tensor([[i * k, i * k + k] for i in range(rows)], **i32)
    if s["masks"] != "none":
        # a grammar allows a few tokens, or nearly all; one of many rows has come to its grammar's end, where none is left
        n = rows if s["masks"] == "all" else -(-rows // 2)
        share = torch.tensor([0.001, 0.02, 0.95])[torch.arange(n) % 3].to(DEV)
        if n >= 8:
            share[5] = 0
        words = -(-vocab // 32)
        mask = torch.zeros(n, words, dtype=torch.int32, device=DEV)
        for b in range(32):                                             # bit b of word w: token 32 w + b
            mask |= (torch.rand(n, words, generator=g, device=DEV) < share[:, None]).int() << b
        s["mask"], s["n_masks"] = mask, n
        s["mask_rows"] = torch.arange(rows, **i32) if s["masks"] == "all" else torch.where(torch.arange(rows, device=DEV) % 2 == 0,
                                                                                           torch.arange(rows, device=DEV) // 2, -1).int()
    s["out_rows"] = torch.empty(rows, vocab, device=DEV)
    s["token"] = torch.empty(rows, **i32)


# ---------------------------------------------------------------- one pass

def run(s):
    if own:
        return _run_own(s)
    return {"norm": _plain_norm, "linear": _plain_linear, "product": _plain_product, "down": _plain_down, "logits": _plain_logits}[s["kind"]](s)


def _run_own(s):
    ud, b, kind, rows = _package(), s["buf"], s["kind"], s["rows"]
    if kind == "logits":
        if "ws" not in b:
            s["ws"] = torch.empty(ud.logits_workspace_bytes(rows, s["vocab"]) + 16, dtype=torch.uint8, device=DEV)
            b["ws"] = Buf(s["ws"])
        ud.logits_process(b["logits"], b["out_rows"], rows, s["vocab"], token=b["token"], tokens=b["tokens"], n_tokens=s["n_tokens"],
                          ranges=b["ranges"], penalties=b["penalties"], bias_ids=b["bias_ids"], bias_values=b["bias_values"],
                          n_biases=rows * s.get("k", 0), bias_ranges=b["bias_ranges"], mask=b["mask"], n_masks=s.get("n_masks", 0),
                          mask_rows=b["mask_rows"], workspace=b["ws"], dtype=s["dtype"])
        return s["out_rows"], s["token"]
    dim, out, dtype = s["dim"], s.get("out"), s["dtype"]
    if kind in ("norm", "linear"):
        eight = kind == "linear"
        ud.rms_norm(b["x"], b["codes"] if eight else b["out_rows"], rows, dim, weight=b["weight"], eps=EPS, residual=b.get("res"), sum_out=b.get("sum"),
                    scales=b["scales"] if eight else None, dtype=dtype, sum_dtype=s["sums"], out_dtype="i8" if eight else dtype)
    if kind == "down":
        ud.i8_quantize(b["up"], b["codes"], b["scales"], rows, dim, gate=b["fused"], dtype=dtype, ld=2 * dim)
    if kind != "norm":
        ud.i8_linear(b["codes"], b["scales"], b["w"], b["w_scales"], b["out_rows"], rows, out, dim, bias=b["bias_row"],
                     residual=b["res"] if kind == "down" else None, dtype=dtype)
    return (s["sum"], s["out_rows"]) if "sum" in s else s["out_rows"]


def _summed(s):
    """What is normed, and the sums as they are stored."""
    if "res" not in s:
        return s["x"].float(), None
    stored = (s["x"].float() + s["res"].float()).to(s["res"].dtype)
    return stored.float(), stored


def _normed(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _eight(y):
    """Rows as int8 codes (in fp32) and their scales."""
    scale = (y.abs().amax(-1, keepdim=True) / 127).clamp(min=TINY)
    return torch.round(y / scale), scale


def _times(s, codes, scale):
    """The product, with its scales and its bias, in fp32."""
    o = torch.matmul(codes, s["w"].float().t()) * scale * s["w_scales"]
    return o if s["bias_row"] is None else o + s["bias_row"]


def _plain_norm(s):
    x, stored = _summed(s)
    y = _normed(x, s["weight"]).to(s["out_rows"].dtype)
    return y if stored is None else (stored, y)


def _plain_linear(s):
    x, stored = _summed(s)
    o = _times(s, *_eight(_normed(x, s["weight"]))).to(s["out_rows"].dtype)
    return o if stored is None else (stored, o)


def _plain_product(s):
    return _times(s, s["codes"].float(), s["scales"][:, None]).to(s["out_rows"].dtype)


def _plain_down(s):
    gate, up = s["fused"].float().split(s["dim"], -1)
    return (_times(s, *_eight(gate / (1 + torch.exp(-gate)) * up)) + s["res"].float()).to(s["out_rows"].dtype)


def _plain_logits(s):
    rows, vocab = s["rows"], s["vocab"]
    x = s["logits"].float()
    at = torch.arange(s["n_tokens"], device=DEV)
    row = torch.bucketize(at, s["ranges"][:, 2].long(), right=True)
    fresh = at >= s["ranges"][row, 1]
    flat = row * vocab + s["tokens"]
    seen = torch.zeros(rows * vocab, device=DEV).index_fill_(0, flat, 1).view(rows, vocab) > 0
    count = torch.zeros(rows * vocab, device=DEV).index_add_(0, flat, fresh.float()).view(rows, vocab)
    rep, pres, freq = s["penalties"].t().unsqueeze(-1).unbind(0)
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (freq * count + pres * (count > 0))
    if s["bias_ids"] is not None:
        at = torch.arange(rows, device=DEV).repeat_interleave(s["k"]) * vocab + s["bias_ids"]
        x = x.view(-1).index_add(0, at, s["bias_values"]).view(rows, vocab)
    if s["mask"] is not None:
        bits = (s["mask"].unsqueeze(-1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        allowed = bits.flatten(1)[:, :vocab][s["mask_rows"].clamp(min=0).long()] > 0
        x = torch.where(allowed | (s["mask_rows"] < 0)[:, None], x, -math.inf)
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device=DEV), vocab).amin(1)
    return x, torch.where(top[:, 0] == -math.inf, -1, first).int()


# ---------------------------------------------------------------- work

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"]
    if case["kind"] == "logits":
        vocab, k = case["vocab"], case["biases"]
        past, new = _spread(case["past"] // 3, case["past"], rows), _spread(case["new"] // 4, case["new"], rows)
        masks = {"none": 0, "some": -(-rows // 2), "all": rows}[case["masks"]]
        return {"bytes": rows * vocab * (size + 4) + masks * vocab // 8 + 4 * sum(past + new) + 8 * rows * k, "flops": 4 * rows * vocab}
    dim, out = case["dim"], case.get("out", 0)
    moved = 0
    if case["kind"] in ("norm", "linear"):
        moved += rows * dim * (size + (2 * (4 if case["sums"] == "f32" else 2) if case["residual"] else 0)) + 4 * dim
    if case["kind"] == "norm":
        return {"bytes": moved + rows * dim * size, "flops": 5 * rows * dim}
    # the rows in 8 bits are written and read between the two calls
    if case["kind"] == "product":
        moved += rows * dim
    elif case["kind"] == "down":
        moved += rows * dim * 2 * size + rows * out * size + 2 * rows * dim
    else:
        moved += 2 * rows * dim
    return {"bytes": moved + out * dim + rows * out * size + 4 * out, "flops": 2 * rows * dim * out}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(s), None
    if case["kind"] == "product":
        return _exact_times(s, s["codes"].double(), s["scales"].double())
    total = None
    if case["kind"] == "down":
        f = s["fused"].double()
        y = f[:, case["dim"]:] * f[:, :case["dim"]] * torch.sigmoid(f[:, :case["dim"]])
    else:
        y = s["x"].double()
        if case["residual"]:
            total = y + s["res"].double()
            y = total.to(s["res"].dtype).double()                       # the norm is that of the sums as they are stored
        y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=1, keepdim=True) ** 2 / case["dim"] + EPS) * s["weight"].double()
    if case["kind"] != "norm":
        scale = torch.clamp(y.abs().max(1).values / 127, min=TINY)
        y = _exact_times(s, torch.round(y / scale[:, None]), scale)
        if case["kind"] == "down":
            y = y + s["res"].double()
    return y if total is None else (total, y)


def _exact_times(s, codes, scale):
    out = torch.empty(len(codes), s["out"], dtype=torch.float64, device=DEV)
    for a in range(0, s["out"], 4096):                                  # sums of whole numbers below 2^53
        w = s["w"][a:a + 4096].double()
        out[:, a:a + 4096] = (codes @ w.T) * torch.outer(scale, s["w_scales"][a:a + 4096].double())
        if s["bias_row"] is not None:
            out[:, a:a + 4096] += s["bias_row"][a:a + 4096].double()
    return out


def _exact_logits(s):
    rows, vocab = s["rows"], s["vocab"]
    out = s["logits"].double()
    for r, (a, b, e) in enumerate(s["ranges"].tolist()):
        rep, pres, freq = s["penalties"][r].double().tolist()
        every = torch.bincount(s["tokens"][a:e].long(), minlength=vocab) > 0
        count = torch.bincount(s["tokens"][b:e].long(), minlength=vocab)
        x = out[r]
        x = torch.where(every & (x > 0), x / rep, torch.where(every, x * rep, x))
        x = x - count * freq - torch.sign(count) * pres
        if s["bias_ids"] is not None:
            a, b = s["bias_ranges"][r].tolist()
            x[s["bias_ids"][a:b].long()] += s["bias_values"][a:b].double()
        if s["mask"] is not None and int(s["mask_rows"][r]) >= 0:
            token = torch.arange(vocab, device=DEV)
            bit = s["mask"][int(s["mask_rows"][r])].long()[token // 32] // 2 ** (token % 32) % 2
            x = x.masked_fill(bit == 0, -math.inf)
        out[r] = x
    return out
