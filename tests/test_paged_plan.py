"""CPU checks of the paged-cache operators' host side: page lists and split plans (csrc/paged_plan.hpp, compiled with the
host compiler) against brute force, the MXFP4 restatement of the tests against an exhaustive search, page sizes, and every
refusal of the calls (none touches the device)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import paged_ref as ref
from conftest import ROOT

SRC = r'''
#include "paged_plan.hpp"
using namespace ud;
extern "C" void list_of(int lo, int hi, int sinks, int* out) { PageList p = page_list(lo, hi, sinks); out[0] = p.sink; out[1] = p.first; out[2] = p.count; }
extern "C" int at(int lo, int hi, int sinks, int u) { return page_at(page_list(lo, hi, sinks), u); }
extern "C" long long most(int span, int sinks) { return max_pages(span, sinks); }
extern "C" void plan(long long want, long long pages, long long step, int* out) {
    SplitPlan p = split_plan(want, pages, step); out[0] = p.splits; out[1] = p.pages; }
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SRC)
    so = str(d / "plan.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "universal-dictator_amd", "csrc"),
                    str(d / "plan.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.most.restype = ctypes.c_longlong
    lib.plan.argtypes = [ctypes.c_longlong] * 3 + [ctypes.c_void_p]
    return lib


def _list(plan, lo, hi, sinks):
    out = (ctypes.c_int * 3)()
    plan.list_of(lo, hi, sinks, out)
    return tuple(out)


def test_page_lists_hold_every_visible_key_once(plan):
    rng = np.random.default_rng(1)
    cases = [(0, 1, 0), (0, 16, 5), (15, 17, 1), (16, 17, 16), (17, 40, 17), (33, 34, 100), (5, 5, 3), (9, 2, 3)]
    cases += [tuple(int(x) for x in (rng.integers(0, 300), rng.integers(0, 400), rng.integers(0, 80))) for _ in range(400)]
    for lo, hi, sinks in cases:
        sink, first, count = _list(plan, lo, hi, sinks)
        pages = [plan.at(lo, hi, sinks, u) for u in range(count)]
        want = sorted({int(j) // 16 for j in ref.visible(lo, hi, sinks, 1 << 30)})
        # window pages run from lo's to (hi - 1)'s; a range inside them is all visible, so the lists agree page for page
        assert pages == want, (lo, hi, sinks)
        if count:
            assert count <= plan.most(hi - lo, sinks)
    top = 2 ** 31 - 1 - 15
    sink, first, count = _list(plan, top - 5, top, 2 ** 31 - 1)
    assert plan.at(top - 5, top, 2 ** 31 - 1, count - 1) == (top - 1) // 16


def test_split_plans_cover_the_list(plan):
    rng = np.random.default_rng(2)
    for _ in range(500):
        want, pages = int(rng.integers(0, 600)), int(rng.integers(1, 20000))
        step = int(rng.choice([1, 8, 16]))
        out = (ctypes.c_int * 2)()
        plan.plan(want, pages, step, out)
        splits, each = out
        assert 1 <= splits <= min(256, max(1, want)) and each % step == 0
        assert splits * each >= pages > (splits - 1) * each


def test_fp4_restatement_is_the_nearest_code():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((200, 64)) * np.exp2(rng.integers(-40, 40, (200, 1)))
    x[0] = 0
    x[1, :32] = [7, 6.9, 6, 5, 5.1, 3.5, 2.5, 1.75, 1.25, .75, .25, .2500001, -.25, -5, -3.5, 0] * 2
    x[2, :32] = 7.0000001
    code, byte = ref.fp4_encode(x)
    y = ref.fp4_decode(code, byte)
    e = np.repeat(byte.astype(np.float64) - 127, 32, -1)
    unit = np.exp2(e)
    best = np.abs(np.abs(x)[..., None] - ref.LEVELS * unit[..., None]).min(-1)
    np.testing.assert_array_equal(np.abs(np.abs(x) - np.abs(y)), best)
    top = np.abs(x).reshape(200, 2, 32).max(-1)
    ok = byte > 27
    assert np.all(top <= 7 * np.exp2(byte.astype(np.float64) - 127))
    assert np.all((top > 7 * np.exp2(byte.astype(np.float64) - 128))[ok])
    assert list(y[1, :16]) == [6, 6, 6, 4, 6, 4, 2, 2, 1, 1, 0, .5, 0, -4, -4, 0]


def test_page_bytes(ud):
    assert ud.kv_page_bytes(8, 128, "bf16") == 8 * 16 * 256
    assert ud.kv_page_bytes(2, 64, "f16") == 2 * 16 * 128
    assert ud.kv_page_bytes(8, 128, "mxfp4") == 8 * 16 * (64 + 4)
    assert ud.kv_page_bytes(3, 64, "mxfp4") == 3 * 16 * (32 + 2)
    lib = ud.load_library()
    for bad in [(3, 8, 128, 16), (1, 0, 128, 16), (1, 8, 96, 16), (1, 8, 128, 32)]:
        assert lib.ud_kv_page_bytes(*bad) == 0


F32, BF16, F16, FP4 = 0, 1, 2, 16
P, ODD = 0x10000, 0x10004                         # pointers that a refused call must not follow


def _refused(ud, name, base, **change):
    """Calls name with base's arguments changed; returns (status, message)."""
    args = dict(base)
    assert set(change) <= set(args)
    args.update(change)
    lib = ud.load_library()
    rc = getattr(lib, name)(*args.values())
    return rc, lib.ud_last_error().decode()


APPEND = dict(dtype=BF16, fmt=BF16, q=P, q_ld=4096, k=P, k_ld=1024, v=P, v_ld=1024, q_out=P, qo_ld=4096, qw=None, kw=None, eps=1e-6,
              inv=None, pos=P, seqs=None, kp=P, vp=P, num=10, bt=P, n=4, max_blocks=9, rows=4, hq=32, hkv=8, d=128, block=16, st=None)
READ = dict(fmt=BF16, dtype=F32, kp=P, vp=P, num=10, bt=P, n=4, max_blocks=9, pos=P, seqs=None, ko=P, vo=P, rows=4, hkv=8, d=128, block=16,
            st=None)
WINDOW = dict(fmt=BF16, dtype=F32, q=P, kp=P, vp=P, num=10, bt=P, max_blocks=9, ranges=P, sinks=4, out=P, n=4, m=1, hq=32, hkv=8, d=128,
              block=16, span=140, ws=P, wsb=1 << 30, st=None)
PREFILL = dict(fmt=BF16, dtype=BF16, q=P, kp=P, vp=P, num=10, bt=P, max_blocks=9, qs=P, ranges=P, sinks=4, out=P, n=4, rows=40, most=20,
               hq=32, hkv=8, d=128, block=16, span=140, ws=P, wsb=1 << 30, st=None)
PAGED = [dict(kp=None), dict(vp=None), dict(bt=None), dict(fmt=F32), dict(fmt=7), dict(d=96), dict(d=256), dict(block=32), dict(n=0),
         dict(n=65536), dict(hkv=0), dict(num=0), dict(max_blocks=0), dict(max_blocks=2 ** 27), dict(kp=ODD), dict(vp=ODD)]


@pytest.mark.parametrize("name,base,changes", [
    ("ud_qk_norm_rope_append", APPEND, [
        dict(k=None), dict(v=None), dict(pos=None), dict(q=None), dict(q_out=None), dict(dtype=F16), dict(dtype=5), dict(rows=-1),
        dict(rows=2 ** 23 + 1), dict(hq=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(q_ld=4095), dict(k_ld=1020), dict(v_ld=1020),
        dict(qo_ld=4092), dict(q_ld=4098), dict(q=0x10004), dict(k=0x10002), dict(dtype=F32, v=0x10008)]),
    ("ud_paged_kv_read", READ, [
        dict(pos=None), dict(ko=None), dict(vo=None), dict(dtype=F16), dict(fmt=FP4, dtype=F16), dict(rows=-1), dict(rows=2 ** 30),
        dict(ko=ODD)]),
    ("ud_gqa_window_attention_paged", WINDOW, [
        dict(q=None), dict(ranges=None), dict(out=None), dict(dtype=F16), dict(dtype=9), dict(m=0), dict(m=9), dict(hq=0), dict(hq=33),
        dict(hq=128, m=5), dict(hq=8 * 65), dict(sinks=-1), dict(span=-1), dict(q=ODD), dict(out=ODD), dict(ws=None), dict(ws=ODD),
        dict(wsb=64), dict(n=65535, m=8, hq=512, hkv=64)]),
    ("ud_gqa_prefill_paged", PREFILL, [
        dict(q=None), dict(qs=None), dict(ranges=None), dict(out=None), dict(dtype=F16), dict(dtype=F32), dict(rows=-1), dict(most=41),
        dict(most=-1), dict(hq=33), dict(hq=8 * 129), dict(sinks=-1), dict(span=-1), dict(q=ODD), dict(out=ODD),
        dict(rows=2 ** 26, most=2 ** 26), dict(span=100000, ws=None), dict(span=100000, wsb=64), dict(span=100000, ws=ODD)]),
])
def test_refusals(ud, name, base, changes):
    """Every refused call returns UD_ERR_INVALID or UD_ERR_SHAPE and names itself."""
    for change in PAGED + changes:
        rc, msg = _refused(ud, name, base, **change)
        assert rc in (-1, -2), (name, change, rc)
        assert msg.startswith(name + ":"), msg


def test_empty_calls_do_nothing(ud):
    assert _refused(ud, "ud_qk_norm_rope_append", APPEND, rows=0)[0] == 0
    assert _refused(ud, "ud_paged_kv_read", READ, rows=0)[0] == 0
    assert _refused(ud, "ud_gqa_prefill_paged", PREFILL, rows=0, most=0)[0] == 0


def test_workspace_sizes(ud):
    """No workspace where one split serves; else room for every split's output, maximum and sum."""
    assert ud.gqa_window_workspace_bytes(1, 1, 32, 8, 128, 0, 100) == 0
    b = ud.gqa_window_workspace_bytes(1, 1, 32, 8, 128, 0, 8192)
    assert b > 0 and b % (32 * 130 * 4) == 0
    assert ud.gqa_window_workspace_bytes(512, 1, 32, 8, 128, 4, 8192) == 0
    assert b <= ud.gqa_window_workspace_bytes(1, 1, 32, 8, 128, 2 ** 31 - 1, 2 ** 31 - 1) <= 256 * 32 * 130 * 4
    assert ud.gqa_prefill_workspace_bytes(64, 6400, 100, 32, 8, 128, 0, 8192) == 0
    assert ud.gqa_prefill_workspace_bytes(1, 20, 20, 32, 8, 128, 0, 100) == 0
    assert ud.gqa_prefill_workspace_bytes(1, 20, 20, 32, 8, 128, 0, 100000) > 0
    for bad in [(0, 1, 32, 8, 128, 0, 100), (1, 0, 32, 8, 128, 0, 100), (1, 1, 32, 0, 128, 0, 100), (1, 1, 32, 8, 128, -1, 100)]:
        assert ud.gqa_window_workspace_bytes(*bad) == 0
