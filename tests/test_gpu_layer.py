"""The calls of include/ud_layer.h together with the paged cache's, as a decoder runs them: a prompt, then tokens one by one, every
step of the layer held against its float64 form on the very values that it was given; the same from replayed graphs and on two
streams."""
import numpy as np
import pytest

import layer_ref as ref
import paged_ref as paged
from test_gpu_rows import GATE_REL, NORM_REL

pytestmark = pytest.mark.gpu

D, HQ, HKV, HD, FF, V, EPS = 512, 8, 4, 64, 1040, 1025, 1e-5
QKV = (HQ + 2 * HKV) * HD


def dev(ud, a):
    return ud.DeviceBuffer.from_numpy(np.ascontiguousarray(a))


class At:
    def __init__(self, buf, off):
        self.ptr, self.nbytes = buf.ptr + off, buf.nbytes - off


class Decoder:
    """One layer and a head, with int8 weights made by i8_quantize on the device, over a paged cache of bf16 pages."""

    def __init__(self, ud, rng, lens):
        self.ud, self.host, self.w = ud, {}, {}
        for name, (n, k) in dict(qkv=(QKV, D), o=(D, HQ * HD), gate_up=(2 * FF, D), down=(D, FF), head=(V, D)).items():
            x = ref.stored(rng.standard_normal((n, k)) * k ** -0.5, "bf16")
            codes, scales = ud.DeviceBuffer(n * k), ud.DeviceBuffer(4 * n)
            ud.i8_quantize(dev(ud, x[0]), codes, scales, n, k)
            ud.synchronize()
            c, s = codes.download((n, k), np.int8), scales.download(n)
            ref.check_codes(c, s.astype(np.float64), x[1], 0.0)
            self.w[name], self.host[name] = (codes, scales), (c, s)
        self.norms = {k: (1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for k in ("one", "two", "last")}
        self.norm_dev = {k: dev(ud, v) for k, v in self.norms.items()}
        self.bias = (0.1 * rng.standard_normal(QKV)).astype(np.float32)
        self.bias_dev = dev(ud, self.bias)
        self.inv = dev(ud, ud.rope_inv_freq(HD))
        self.table, self.num = paged.assign_pages(rng, lens)
        self.n, self.most = self.table.shape
        self.bt = dev(ud, self.table)
        self.pages = [dev(ud, np.zeros(self.num * HKV * 16 * HD, np.uint16)) for _ in range(2)]

    def buffers(self, rows):
        ud = self.ud
        size = dict(x=2 * rows * D, res=4 * rows * D, sum1=4 * rows * D, sum2=4 * rows * D, c1=rows * D, s1=4 * rows, qkv=2 * rows * QKV,
                    q=2 * rows * HQ * HD, att=2 * rows * HQ * HD, c2=rows * HQ * HD, s2=4 * rows, o=2 * rows * D, c3=rows * D, s3=4 * rows,
                    gu=4 * rows * FF, c4=rows * FF, s4=4 * rows, down=2 * rows * D, sum3=4 * rows * D, c5=rows * D, s5=4 * rows, logits=4 * rows * V,
                    out=4 * rows * V, token=4 * rows, ws=ud.logits_workspace_bytes(rows, V))
        return {k: ud.DeviceBuffer(v) for k, v in size.items()}

    def linear(self, name, codes, scales, out, rows, stream, **kw):
        n, k = self.host[name][0].shape
        self.ud.i8_linear(codes, scales, *self.w[name], out, rows, n, k, hip_stream=stream, **kw)

    def run(self, b, rows, plan, stream=None):
        """From x (bf16) and res (fp32), both [rows, D], to a token for each row."""
        ud, st = self.ud, dict(hip_stream=stream)
        ud.rms_norm(b["x"], b["c1"], rows, D, weight=self.norm_dev["one"], eps=EPS, residual=b["res"], sum_out=b["sum1"], scales=b["s1"],
                    sum_dtype="f32", out_dtype="i8", **st)
        self.linear("qkv", b["c1"], b["s1"], b["qkv"], rows, stream, bias=self.bias_dev)
        k, v = At(b["qkv"], 2 * HQ * HD), At(b["qkv"], 2 * (HQ + HKV) * HD)
        ud.qk_norm_rope_append(b["qkv"], k, v, b["q"], *self.pages, self.num, self.bt, self.n, self.most, plan["pos"], rows, HQ, HKV, HD,
                               seqs=plan["seqs"], inv_freq=self.inv, q_ld=QKV, k_ld=QKV, v_ld=QKV, **st)
        if "q_start" in plan:
            ud.gqa_prefill_paged(b["q"], *self.pages, self.num, self.bt, self.most, plan["q_start"], plan["ranges"], 0, b["att"], self.n, rows,
                                 plan["longest"], HQ, HKV, HD, plan["span"], plan["ws"], **st)
        else:
            ud.gqa_window_attention_paged(b["q"], *self.pages, self.num, self.bt, self.most, plan["ranges"], 0, b["att"], self.n, 1, HQ, HKV, HD,
                                          plan["span"], plan["ws"], dtype="bf16", **st)
        ud.i8_quantize(b["att"], b["c2"], b["s2"], rows, HQ * HD, **st)
        self.linear("o", b["c2"], b["s2"], b["o"], rows, stream)
        ud.rms_norm(b["o"], b["c3"], rows, D, weight=self.norm_dev["two"], eps=EPS, residual=b["sum1"], sum_out=b["sum2"], scales=b["s3"],
                    sum_dtype="f32", out_dtype="i8", **st)
        self.linear("gate_up", b["c3"], b["s3"], b["gu"], rows, stream)
        ud.i8_quantize(At(b["gu"], 2 * FF), b["c4"], b["s4"], rows, FF, gate=b["gu"], ld=2 * FF, **st)
        self.linear("down", b["c4"], b["s4"], b["down"], rows, stream, residual=b["o"])
        ud.rms_norm(b["down"], b["c5"], rows, D, weight=self.norm_dev["last"], eps=EPS, residual=b["sum2"], sum_out=b["sum3"], scales=b["s5"],
                    sum_dtype="f32", out_dtype="i8", **st)
        self.linear("head", b["c5"], b["s5"], b["logits"], rows, stream, dtype="f32")
        ud.logits_process(b["logits"], b["out"], rows, V, token=b["token"], tokens=plan["tokens"], n_tokens=plan["n_tokens"],
                          ranges=plan["histories"], penalties=plan["penalties"], mask=plan["mask"], n_masks=1, mask_rows=plan["mask_rows"],
                          workspace=b["ws"], **st)

    def plan(self, new, past, histories, rng):
        """The arrays of a pass over new[i] rows of each sequence behind past[i]."""
        ud, rows = self.ud, sum(new)
        pos = np.concatenate([p + np.arange(m) for p, m in zip(past, new)])
        seqs = np.repeat(np.arange(self.n), new)
        span = max(p + m for p, m in zip(past, new))
        at = np.concatenate([[0], np.cumsum([len(h) for h in histories])])
        hist = np.array([[at[i], at[i] + len(histories[i]) // 2, at[i + 1]] for i in seqs], np.int32)
        allowed = rng.random((1, V)) < 0.5
        p = dict(pos=dev(ud, pos.astype(np.int32)), seqs=dev(ud, seqs.astype(np.int32)), span=span,
                 ranges=dev(ud, np.stack([np.zeros_like(pos), pos + 1], 1).astype(np.int32)),
                 tokens=dev(ud, np.concatenate(histories).astype(np.int32)), n_tokens=int(at[-1]), histories=dev(ud, hist),
                 penalties=dev(ud, np.tile(np.array([[1.2, 0.3, 0.1]], np.float32), (rows, 1))), mask=dev(ud, ref.mask_words(allowed)),
                 mask_rows=dev(ud, np.where(seqs == 0, 0, -1).astype(np.int32)))
        p["host"] = dict(tokens=np.concatenate(histories).astype(np.int32), hist=hist, pen=np.tile(np.array([[1.2, 0.3, 0.1]], np.float32), (rows, 1)),
                         masks=[allowed[0] if s == 0 else None for s in seqs])
        if max(new) > 1:
            p.update(q_start=dev(ud, np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), longest=max(new))
            need = ud.gqa_prefill_workspace_bytes(self.n, rows, max(new), HQ, HKV, HD, 0, span)
        else:
            need = ud.gqa_window_workspace_bytes(self.n, 1, HQ, HKV, HD, 0, span)
        p["ws"] = ud.DeviceBuffer(need) if need else None
        return p

    def check(self, b, rows, plan):
        """Each step against its float64 form, on the step's own inputs as they lie in memory."""
        f32 = lambda k, w: b[k].download((rows, w)).astype(np.float64)  # noqa: E731
        b16 = lambda k, w: ref.from_bits(b[k].download((rows, w), np.uint16), "bf16")  # noqa: E731
        codes = lambda k, w: b[k].download((rows, w), np.int8)  # noqa: E731
        scales = lambda k: b[k].download(rows).astype(np.float64)  # noqa: E731

        def normed(x, res, total, weight, c, s):
            np.testing.assert_array_equal(f32(total, D), ref.summed(b16(x, D), f32(res, D), "f32"))
            ref.check_codes(codes(c, D), scales(s), ref.normed(f32(total, D), self.norms[weight], float(np.float32(EPS))), NORM_REL)

        def product(name, c, s, got, dtype, bias=None, residual=None):
            w, ws = self.host[name]
            want, mag = ref.product(codes(c, w.shape[1]), scales(s), w, ws, bias, residual)
            assert np.all(np.abs(got - want) <= 5.05 * ref.STEP32 * mag + 1.01 * ref.HALF_STEP[dtype] * np.abs(want))

        normed("x", "res", "sum1", "one", "c1", "s1")
        product("qkv", "c1", "s1", b16("qkv", QKV), "bf16", bias=self.bias)
        att = b16("att", HQ * HD)
        assert np.all(np.isfinite(att)) and np.all(np.abs(att).max(1) > 0)
        ref.check_codes(codes("c2", HQ * HD), scales("s2"), att, 0.0)
        product("o", "c2", "s2", b16("o", D), "bf16")
        normed("o", "sum1", "sum2", "two", "c3", "s3")
        gu = b16("gu", 2 * FF)
        product("gate_up", "c3", "s3", gu, "bf16")
        ref.check_codes(codes("c4", FF), scales("s4"), ref.gated(gu[:, FF:], gu[:, :FF]), GATE_REL)
        product("down", "c4", "s4", b16("down", D), "bf16", residual=b16("o", D))
        normed("down", "sum2", "sum3", "last", "c5", "s5")
        logits = f32("logits", V)
        product("head", "c5", "s5", logits, "f32")
        h = plan["host"]
        want, mag = ref.logits_out(logits, h["tokens"], h["hist"], h["pen"], None, h["masks"])
        out = f32("out", V)
        np.testing.assert_array_equal(np.isinf(out), np.isinf(want))
        fine = np.isfinite(want)
        assert np.all(np.abs(out[fine] - want[fine]) <= 5.05 * ref.STEP32 * mag[fine])
        token = b["token"].download(rows, np.int32)
        np.testing.assert_array_equal(token, ref.chosen(out))
        return token


def embed(rng, b, table, tokens):
    rows = len(tokens)
    b["x"].upload(ref.stored(table[tokens % len(table)], "bf16")[0])
    b["res"].upload((0.5 * rng.standard_normal((rows, D))).astype(np.float32))


def test_prompt_and_tokens(gpu):
    ud, rng = gpu, np.random.default_rng(11)
    lens = [61, 30]
    m = Decoder(ud, rng, lens)
    table = rng.standard_normal((V, D))
    new, past = [43, 21], [0, 0]
    histories = [rng.integers(0, V, 40), rng.integers(0, V, 9)]
    for step in range(5):
        rows = sum(new)
        b, p = m.buffers(rows), m.plan(new, past, histories, rng)
        embed(rng, b, table, rng.integers(0, V, rows) if step == 0 else np.array([h[-1] for h in histories]))
        m.run(b, rows, p)
        ud.synchronize()
        token = m.check(b, rows, p)
        last = np.cumsum(new) - 1
        histories = [np.append(h, token[i]) for h, i in zip(histories, last)]
        past = [a + c for a, c in zip(past, new)]
        new = [1, 1]


def test_steps_in_replayed_graphs(gpu):
    """A token's step captured once: every replay gives the eager run's bits, with other work and waits between, from two graphs that
    share their buffers and workspaces."""
    ud, rng = gpu, np.random.default_rng(12)
    m = Decoder(ud, rng, [40, 40])
    table = rng.standard_normal((V, D))
    histories = [rng.integers(0, V, 30), rng.integers(0, V, 60)]
    b, p = m.buffers(2), m.plan([1, 1], [25, 7], histories, rng)
    keep = ["sum3", "gu", "logits", "out", "token", "c4", "s4"]
    read = lambda: {k: b[k].download(b[k].nbytes, np.uint8) for k in keep}  # noqa: E731
    other, po = m.buffers(2), m.plan([1, 1], [38, 39], histories, rng)
    stream = ud.HipStream()
    graphs = []
    for _ in range(2):
        with ud.Graph.capture(stream) as g:
            m.run(b, 2, p, stream)
        graphs.append(g)
    for turn in range(4):
        embed(rng, b, table, rng.integers(0, V, 2))
        embed(rng, other, table, rng.integers(0, V, 2))
        m.run(b, 2, p, stream)
        stream.synchronize()
        m.check(b, 2, p)
        want = read()
        for g in graphs:
            for k in keep:
                ud._check(ud.lib().ud_memset(b[k].ptr, 0x5A, b[k].nbytes))
            m.run(other, 2, po, stream)
            g.launch(stream)
            stream.synchronize()
            got = read()
            for k in keep:
                np.testing.assert_array_equal(got[k], want[k], err_msg="%s, turn %d" % (k, turn))


def test_two_streams(gpu):
    """Products, rows and logits of two streams at once, each with its own buffers, many times over."""
    ud = gpu
    rng = np.random.default_rng(13)
    m = Decoder(ud, rng, [40, 40])
    table = rng.standard_normal((V, D))
    histories = [rng.integers(0, V, 3000), rng.integers(0, V, 60)]
    streams, sets = [ud.HipStream() for _ in range(2)], []
    for i in range(2):
        mine = Decoder.__new__(Decoder)
        mine.__dict__.update(m.__dict__)
        mine.pages = [dev(ud, np.zeros(m.num * HKV * 16 * HD, np.uint16)) for _ in range(2)]
        b, p = m.buffers(2), m.plan([1, 1], [3 + i, 7], histories, rng)
        embed(rng, b, table, rng.integers(0, V, 2))
        mine.run(b, 2, p)
        ud.synchronize()
        mine.check(b, 2, p)
        sets.append((mine, b, p, b["out"].download((2, V)), b["sum3"].download((2, D))))
    for _ in range(20):
        for s, (mine, b, p, _, _) in zip(streams, sets):
            mine.run(b, 2, p, s)
    ud.synchronize()
    for mine, b, p, out, total in sets:
        np.testing.assert_array_equal(b["out"].download((2, V)), out)
        np.testing.assert_array_equal(b["sum3"].download((2, D)), total)


@pytest.mark.parametrize("N,K", [(1000, 4096), (6144, 1024), (520, 8208)])
def test_rows_do_not_depend_on_the_batch(gpu, N, K):
    """A row's product, norm and 8-bit codes are the same bits alone and in batches that take other kernels; a repeated call's too."""
    ud, rng = gpu, np.random.default_rng([N, K])
    most = 700
    x, _ = ref.stored(rng.standard_normal((most, K)), "bf16")
    w = rng.integers(-127, 128, (N, K)).astype(np.int8)
    wd, wsd, xd = dev(ud, w), dev(ud, rng.uniform(0.5, 2, N).astype(np.float32) * 1e-3), dev(ud, x)
    c, s, o = ud.DeviceBuffer(most * K), ud.DeviceBuffer(4 * most), ud.DeviceBuffer(4 * most * N)
    bias, res = dev(ud, rng.standard_normal(N).astype(np.float32)), dev(ud, rng.standard_normal((most, N)).astype(np.float32))

    def go(rows):
        ud.rms_norm(xd, c, rows, K, scales=s, out_dtype="i8")
        got = []
        for kw in (dict(), dict(bias=bias, residual=res)):
            ud.i8_linear(c, s, wd, wsd, o, rows, N, K, dtype="f32", **kw)
            ud.synchronize()
            got.append(o.download((rows, N)))
        return c.download((rows, K), np.int8), s.download(rows), *got

    want = go(most)
    for rows in (1, 3, 16, 17, 40, 100, 300, most):
        for a, e in zip(go(rows), want):
            np.testing.assert_array_equal(a, e[:rows])
