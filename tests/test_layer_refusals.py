"""CPU checks of the calls of include/ud_layer.h: every refusal (none touches the device), calls over nothing, the size of the
workspace, and the overlap rule (csrc/layer.hpp) against brute force."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from conftest import ROOT

P = 1 << 20                            # an aligned address that is never read
F32, BF16, F16, I8 = 0, 1, 2, 32


def refused(ud, rc, *words):
    lib = ud.load_library()
    assert rc < 0, rc
    msg = lib.ud_last_error().decode()
    for w in words:
        assert w in msg, msg


def norm(ud, **kw):
    a = dict(dtype=BF16, x=P, x_ld=64, sum_dtype=BF16, res=None, sum=None, sum_ld=64, w=None, eps=1e-6, out_dtype=BF16, out=2 * P, out_ld=64,
             scales=None, rows=4, dim=64)
    a.update(kw)
    return ud.load_library().ud_rms_norm(a["dtype"], a["x"], a["x_ld"], a["sum_dtype"], a["res"], a["sum"], a["sum_ld"], a["w"], a["eps"],
                                         a["out_dtype"], a["out"], a["out_ld"], a["scales"], a["rows"], a["dim"], None)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(dtype=I8), dict(out_dtype=F32), dict(out_dtype=7), dict(rows=-1), dict(rows=1 << 22), dict(dim=0), dict(dim=12),
    dict(dim=32776, x_ld=32776, out_ld=32776), dict(x_ld=56), dict(x_ld=68), dict(out_ld=60), dict(x=None), dict(out=None), dict(x=P + 8),
    dict(out=2 * P + 8), dict(w=P + 4), dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(scales=3 * P),
    dict(out_dtype=I8), dict(out_dtype=I8, scales=3 * P + 2), dict(out_dtype=I8, scales=3 * P, out=2 * P + 4),
    dict(res=3 * P), dict(sum=3 * P), dict(res=3 * P, sum=4 * P, sum_dtype=F16), dict(res=3 * P, sum=4 * P, sum_ld=56),
    dict(res=3 * P + 8, sum=4 * P), dict(res=3 * P, sum=4 * P + 8), dict(res=3 * P, sum=4 * P, sum_ld=68),
    # overlaps
    dict(out=P + 16), dict(out=P, out_ld=72), dict(out=P, out_dtype=I8, scales=3 * P), dict(res=3 * P, sum=3 * P + 128),
    dict(res=3 * P, sum=P, sum_dtype=F32), dict(res=3 * P, sum=2 * P), dict(res=3 * P, sum=2 * P + 256), dict(out=3 * P, res=3 * P + 16, sum=4 * P),
    dict(out_dtype=I8, scales=P + 64), dict(out_dtype=I8, scales=2 * P + 252), dict(w=2 * P + 64), dict(res=3 * P, sum=4 * P, w=4 * P),
    dict(out_dtype=I8, out=2 * P, scales=3 * P, res=3 * P, sum=3 * P),
])
def test_norm_refusals(ud, kw):
    refused(ud, norm(ud, **kw), "ud_rms_norm")


def quantize(ud, **kw):
    a = dict(dtype=BF16, x=P, gate=None, ld=64, codes=2 * P, codes_ld=64, scales=3 * P, rows=4, dim=64)
    a.update(kw)
    return ud.load_library().ud_i8_quantize(a["dtype"], a["x"], a["gate"], a["ld"], a["codes"], a["codes_ld"], a["scales"], a["rows"], a["dim"], None)


@pytest.mark.parametrize("kw", [
    dict(dtype=5), dict(rows=-1), dict(rows=1 << 22), dict(dim=4), dict(dim=65), dict(dim=40000, ld=40000, codes_ld=40000), dict(ld=56), dict(ld=65),
    dict(codes_ld=63), dict(codes_ld=68), dict(x=None), dict(codes=None), dict(scales=None), dict(x=P + 2), dict(gate=4 * P + 8),
    dict(codes=2 * P + 4), dict(scales=3 * P + 1), dict(codes=P), dict(codes=P + 496), dict(gate=4 * P, codes=4 * P), dict(scales=P + 4),
    dict(scales=2 * P + 64), dict(gate=4 * P, scales=4 * P + 508),
])
def test_quantize_refusals(ud, kw):
    refused(ud, quantize(ud, **kw), "ud_i8_quantize")


def linear(ud, **kw):
    a = dict(dtype=BF16, codes=P, codes_ld=64, scales=2 * P, w=3 * P, w_ld=64, w_scales=4 * P, bias=None, res=None, res_ld=40, out=5 * P, out_ld=40,
             M=4, N=40, K=64)
    a.update(kw)
    return ud.load_library().ud_i8_linear(a["dtype"], a["codes"], a["codes_ld"], a["scales"], a["w"], a["w_ld"], a["w_scales"], a["bias"], a["res"],
                                          a["res_ld"], a["out"], a["out_ld"], a["M"], a["N"], a["K"], None)


@pytest.mark.parametrize("kw", [
    dict(dtype=I8), dict(M=-1), dict(M=1 << 22), dict(N=0), dict(N=(1 << 24) + 1, out_ld=1 << 25), dict(M=1 << 20, N=(1 << 18) + 1, out_ld=1 << 19), dict(codes_ld=(1 << 22) + 16), dict(w_ld=1 << 23), dict(K=0), dict(K=8), dict(K=72, codes_ld=80, w_ld=80),
    dict(K=131072, codes_ld=131072, w_ld=131072), dict(codes_ld=48), dict(codes_ld=72), dict(w_ld=56), dict(w_ld=68), dict(out_ld=39),
    dict(res=6 * P, res_ld=39), dict(codes=None), dict(scales=None), dict(w=None), dict(w_scales=None), dict(out=None), dict(codes=P + 8),
    dict(w=3 * P + 4), dict(scales=2 * P + 2), dict(w_scales=4 * P + 1), dict(bias=6 * P + 2), dict(out=5 * P + 1), dict(res=6 * P + 1),
    dict(dtype=F32, out=5 * P + 2),
    # overlaps
    dict(out=P + 16), dict(out=3 * P), dict(out=3 * P + 40 * 64 - 2), dict(out=2 * P), dict(out=4 * P + 158), dict(bias=6 * P, out=6 * P + 40),
    dict(res=5 * P + 2), dict(res=5 * P, res_ld=48), dict(res=5 * P + 80),
])
def test_linear_refusals(ud, kw):
    refused(ud, linear(ud, **kw), "ud_i8_linear")


def logits(ud, **kw):
    a = dict(dtype=F32, x=P, ld=100, out=2 * P, out_ld=100, token=3 * P, n=4, vocab=100, tokens=None, n_tokens=0, ranges=None, pen=None, ids=None,
             vals=None, n_biases=0, br=None, mask=None, mask_ld=4, n_masks=4, rows=None, ws=4 * P, ws_bytes=1 << 16)
    a.update(kw)
    return ud.load_library().ud_logits_process(a["dtype"], a["x"], a["ld"], a["out"], a["out_ld"], a["token"], a["n"], a["vocab"], a["tokens"],
                                               a["n_tokens"], a["ranges"], a["pen"], a["ids"], a["vals"], a["n_biases"], a["br"], a["mask"],
                                               a["mask_ld"], a["n_masks"], a["rows"], a["ws"], a["ws_bytes"], None)


HIST = dict(tokens=5 * P, n_tokens=64, ranges=6 * P, pen=7 * P)
BIAS = dict(ids=8 * P, vals=9 * P, n_biases=64, br=10 * P)


@pytest.mark.parametrize("kw", [
    dict(dtype=9), dict(n=-1), dict(n=65536), dict(vocab=0), dict(vocab=(1 << 24) + 1, ld=1 << 25, out_ld=1 << 25), dict(ld=99), dict(out_ld=99),
    dict(n_tokens=-1), dict(n_biases=-1), dict(mask=11 * P, mask_ld=3), dict(mask=11 * P, n_masks=3), dict(mask=11 * P, n_masks=-1, rows=12 * P),
    dict(x=None), dict(out=None), dict(tokens=5 * P, n_tokens=4), dict(ids=8 * P, vals=9 * P, n_biases=1), dict(ids=8 * P, br=9 * P, n_biases=1),
    dict(ws=None), dict(ws_bytes=31), dict(ws=4 * P + 4), dict(x=P + 2), dict(dtype=BF16, x=P + 1), dict(out=2 * P + 2), dict(token=3 * P + 2),
    dict(HIST, tokens=5 * P + 1), dict(HIST, ranges=6 * P + 2), dict(HIST, pen=7 * P + 1), dict(BIAS, ids=8 * P + 2), dict(BIAS, vals=9 * P + 2),
    dict(BIAS, br=10 * P + 2), dict(mask=11 * P + 2), dict(mask=11 * P, rows=12 * P + 2),
    # overlaps
    dict(out=P, dtype=BF16), dict(out=P + 4), dict(out=P, out_ld=104), dict(token=P), dict(token=2 * P + 8), dict(ws=P), dict(ws=2 * P), dict(ws=3 * P + 8),
    dict(HIST, out=5 * P), dict(HIST, token=5 * P + 128), dict(HIST, ws=7 * P), dict(HIST, token=6 * P), dict(BIAS, out=8 * P), dict(BIAS, token=9 * P),
    dict(BIAS, ws=10 * P), dict(mask=11 * P, out=11 * P + 32), dict(mask=11 * P, rows=12 * P, token=12 * P),
])
def test_logits_refusals(ud, kw):
    refused(ud, logits(ud, **kw), "ud_logits_process")


def test_nothing_to_do(ud):
    """No rows: accepted, and the pointers may be anything."""
    assert norm(ud, rows=0, x=None, out=None) == 0
    assert quantize(ud, rows=0, x=None, codes=None, scales=None) == 0
    assert linear(ud, M=0, codes=None, w=None, scales=None, w_scales=None, out=None) == 0
    assert logits(ud, n=0, x=None, out=None, token=None) == 0


def test_workspace_bytes(ud):
    f = ud.logits_workspace_bytes
    assert f(0, 100) == 0 and f(1, 0) == 0 and f(65536, 10) == 0 and f(1, (1 << 24) + 1) == 0
    for n, v in [(1, 1), (1, 131072), (64, 131072), (65535, 8193), (3, 1 << 24)]:
        assert f(n, v) >= 8 * n * -(-v // 32768)              # a segment has 32,768 tokens at most




def test_overlap_rule(tmp_path):
    """The host part of layer.hpp alone, against the sets of bytes."""
    text = open(os.path.join(ROOT, "universal-dictator_amd", "csrc", "layer.hpp")).read()
    block = re.search(r"struct Block \{.*?\n\};\n", text, re.S).group(0)
    fn = re.search(r"static inline bool blocks_meet.*?\n\}\n", text, re.S).group(0)
    (tmp_path / "m.cpp").write_text("#include <cstdint>\n" + block + fn + r'''
extern "C" int meet(long long at, long long lda, long long wa, long long ra, long long bt, long long ldb, long long wb, long long rb) {
    return blocks_meet(Block{(const void*)at, lda, wa, ra}, Block{(const void*)bt, ldb, wb, rb}); }
''')
    so = str(tmp_path / "m.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(tmp_path / "m.cpp"), "-o", so], check=True)
    f = ctypes.CDLL(so).meet
    f.argtypes = [ctypes.c_longlong] * 8
    rng = np.random.default_rng(1)
    for _ in range(20000):
        ld = int(rng.integers(1, 12))
        same = rng.random() < 0.7
        a = [1000 + int(rng.integers(0, 60)), ld, int(rng.integers(1, 13)), int(rng.integers(1, 5))]
        b = [1000 + int(rng.integers(0, 60)), ld if same else int(rng.integers(1, 12)), int(rng.integers(1, 13)), int(rng.integers(1, 5))]
        at = lambda x: {x[0] + i * x[1] + j for i in range(x[3]) for j in range(x[2])}  # noqa: E731
        truth = bool(at(a) & at(b))
        got = bool(f(*a, *b))
        exact = a[1] == b[1] or a[3] == 1 or b[3] == 1
        assert got == truth if exact else got or not truth, (a, b)
