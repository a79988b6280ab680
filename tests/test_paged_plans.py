"""CPU checks of the windowed and prompt attention's plans (csrc/paged_plan.hpp, compiled with the host compiler): no plan needs
more than the workspace that the caller is told to bring, every workgroup's place is launched, the order by length takes each
sequence once, and the sizes of tests/test_gpu_paged_plans.py reach the paths that they are there for."""
import ctypes
import itertools
import os
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from test_gpu_paged_plans import BY_LENGTH, LONG, SPAN

SRC = r'''
#include "paged_plan.hpp"
using namespace ud;
extern "C" void window(int fp4, int rows, int n, int kv, int sinks, int span, int* o) {
    const WindowPlan p = window_plan(fp4, rows, n, kv, sinks, span);
    o[0] = p.split.splits; o[1] = p.split.pages; o[2] = p.waves; o[3] = p.tiles; o[4] = p.groups; o[5] = p.layer; }
extern "C" int most(int n, int kv, int sinks, int span) { return window_most_splits(n, kv, sinks, span); }
extern "C" int key(int length, int seq) { return length_key(length, seq); }
extern "C" int rank(int z, int layer, int n) { return rank_of_layer(z, layer, n); }
extern "C" int prompt(int n, int kv, int rows, int group, int sinks, int span) {
    return prefill_splits(n, kv, prefill_blocks(rows, group), sinks, span); }
// the first (units, pages) up to the given ones whose finest plan is not the one that the workspace is made for; 0: none
extern "C" int finer(int units, int pages) {
    for (int u = 1; u <= units; u++)
        for (int p = 1; p <= pages; p += 1 + p / 50) {
            const int most = window_most_splits(u, 1, 0, 16 * p);
            for (int fp4 = 0; fp4 < 2; fp4++)
                for (int rows : {1, 16, 17, 64})
                    if (window_plan(fp4, rows, u, 1, 0, 16 * p).split.splits > most) return u;
        }
    return 0; }
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plans")
    (d / "plans.cpp").write_text(SRC)
    so = str(d / "plans.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "universal-dictator_amd", "csrc"),
                    str(d / "plans.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


def _window(plan, *a):
    o = (ctypes.c_int * 6)()
    plan.window(*a, o)
    return dict(zip(("splits", "pages", "waves", "tiles", "groups", "layer"), o))


def test_no_plan_needs_more_than_the_workspace(plan):
    assert plan.finer(1200, 9000) == 0
    rng = np.random.default_rng(1)
    for _ in range(3000):
        n, kv = int(2 ** rng.uniform(0, 16)), int(2 ** rng.uniform(0, 8))
        sinks, span = (int(2 ** rng.uniform(0, 31)) - 1 for _ in range(2))
        n = min(n, 65535)
        for fp4, rows in itertools.product((0, 1), (1, 16, 17, 64)):
            p = _window(plan, fp4, rows, n, kv, sinks, span)
            assert 1 <= p["splits"] <= plan.most(n, kv, sinks, span) <= 256, (fp4, rows, n, kv, sinks, span)


def test_workspace_bytes_hold_the_most_splits(plan, ud):
    for n, m, hq, kv, d, sinks, span in [(1, 1, 32, 8, 128, 0, 8192), (3, 4, 28, 4, 64, 20, 50_000), (64, 1, 32, 8, 128, 4, 4096), (1, 8, 8, 1, 64, 0, 200_000)]:
        s = plan.most(n, kv, sinks, span)
        assert ud.gqa_window_workspace_bytes(n, m, hq, kv, d, sinks, span) == (0 if s == 1 else n * m * hq * s * (d + 2) * 4)
    for n, rows, most, hq, kv, d, sinks, span in [(1, 16, 16, 32, 8, 128, 0, 16_016), (6, 1800, 563, 32, 8, 128, 0, 12_563), (2, 40, 30, 4, 4, 64, 9, 3000)]:
        s = plan.prompt(n, kv, most, hq // kv, sinks, span)
        assert ud.gqa_prefill_workspace_bytes(n, rows, most, hq, kv, d, sinks, span) == (0 if s == 1 else rows * hq * s * (d + 2) * 4)


def test_workgroups_cover_the_rows(plan):
    """Eight waves only for one tile of rows over 16-bit pages (the kernels that there are); the groups' tiles hold all rows."""
    for fp4, rows, n, kv, span in itertools.product((0, 1), range(1, 65), (1, 7, 40, 64, 500), (1, 8), (100, 3000, 100_000)):
        p = _window(plan, fp4, rows, n, kv, 0, span)
        assert p["waves"] in (4, 8) and p["tiles"] in (1, 2)
        assert p["waves"] == 4 or (not fp4 and p["tiles"] == p["groups"] == 1)
        assert p["groups"] * 16 * p["tiles"] >= rows > (p["groups"] - 1) * 16 * p["tiles"]
        assert p["pages"] % (p["waves"] * (4 if fp4 else 2)) == 0


def test_the_order_by_length_takes_each_sequence_once(plan):
    rng = np.random.default_rng(2)
    for n in range(1, 65):
        for layer in {1, 2, n // 2 + 1, n}:
            ranks = [plan.rank(z, layer, n) for z in range(n)]
            assert sorted(ranks) == list(range(n)) and ranks[:layer] == list(range(min(layer, n)))
            assert ranks[layer:] == list(range(n - 1, layer - 1, -1))
        lens = [int(x) for x in rng.choice([0, -5, 3, 3, 2 ** 25, 2 ** 31 - 16, 77], n)]
        keys = [plan.key(L, i) for i, L in enumerate(lens)]
        assert len(set(keys)) == n and min(keys) >= 0 and max(keys) < 2 ** 31
        order = sorted(range(n), key=lambda i: -keys[i])
        held = [min(max(lens[i], 0), 2 ** 25 - 1) for i in order]
        assert held == sorted(held, reverse=True)


def test_only_batches_that_fit_a_wave_are_ranked(plan):
    for fp4, rows, n, kv, span in itertools.product((0, 1), (1, 16, 17, 33, 64), (1, 2, 33, 50, 64, 65, 1000), (1, 6, 8, 200, 300), (2000, 2048, 9000)):
        p = _window(plan, fp4, rows, n, kv, 0, span)
        assert 0 <= p["layer"] <= n
        if p["layer"]:
            assert n <= 64 and n * kv > 256 and p["splits"] == 1 and span > 2032


@pytest.mark.parametrize("fmt,dtype,n,hkv,group,M,layer", BY_LENGTH)
def test_sizes_of_the_batches_by_length(plan, fmt, dtype, n, hkv, group, M, layer):
    p = _window(plan, fmt == "mxfp4", group * M, n, hkv, 0, SPAN)
    assert p["splits"] == 1 and p["layer"] == layer
    assert fmt != "mxfp4" or n - layer > 4


def test_sizes_of_the_long_sequences(plan):
    for fmt, dtype, d, hq, keys, splits in LONG:
        assert _window(plan, fmt == "mxfp4", hq, 1, 1, 0, keys)["splits"] == splits > 64, (fmt, hq, keys)
    assert {_window(plan, f == "mxfp4", h, 1, 1, 0, k)["waves"] for f, _, _, h, k, _ in LONG} == {4, 8}
