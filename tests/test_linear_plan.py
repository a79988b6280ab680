"""CPU check of the int8 product's choice of kernels (csrc/linear_plan.hpp, compiled with the host compiler): every kernel is
chosen for some sizes, the sizes that the GPU tests take reach every one of them, and no choice launches too many threads."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import test_gpu_i8_linear as gpu_tests
from conftest import ROOT

NAMES = ["few 16x16", "few 16x16 deep", "few 16x16 short", "split 16x16", "split 16x32", "split 32x32", "split 64x32", "64x64", "64x128", "128x64", "128x128", "128x128 two", "256x192", "256x256"]
TILE = [(16, 16), (16, 16), (16, 16), (16, 16), (16, 32), (32, 32), (64, 32), (64, 64), (64, 128), (128, 64), (128, 128), (128, 128), (256, 192), (256, 256)]
THREADS = [256, 512, 256, 512] + 9 * [256] + [512]


@pytest.fixture(scope="module")
def kernel(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text('#include "linear_plan.hpp"\nextern "C" int pick(long long M, long long N, long long K) '
                                '{ return (int)ud::linear_kernel(M, N, K); }\nextern "C" int count() { return ud::LINEAR_KERNELS; }\n')
    so = str(d / "plan.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "universal-dictator_amd", "csrc"),
                    str(d / "plan.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.pick.argtypes = [ctypes.c_longlong] * 3
    assert lib.count() == len(NAMES)
    return lib.pick


def test_gpu_tests_reach_every_kernel(kernel):
    seen = {NAMES[kernel(*s)] for s in gpu_tests.TILES + [(M, 515, 1040) for M in gpu_tests.ROWS]}
    assert seen == set(NAMES), set(NAMES) - seen


def test_launches_stay_small(kernel):
    rng = np.random.default_rng(1)
    sizes = [((1 << 22) - 1, 1 << 16, 16), (1 << 14, 1 << 24, 131056), (4, 1 << 24, 8192), (5, 1 << 24, 64), ((1 << 22) - 1, 1, 16), ((1 << 22) - 1, 65536, 131056), (64, 1 << 24, 64),
             (65, 1 << 24, 64), (300, 1 << 24, 64)]
    sizes += [tuple(int(x) for x in np.exp(rng.uniform(0, [15.2, 16.6, 11.7]))) for _ in range(20000)]
    for M, N, K in sizes:
        M, N, K = max(1, M), max(1, min(N, (1 << 38) // max(1, M))), max(16, K // 16 * 16)
        k = kernel(M, N, K)
        tm, tn = TILE[k]
        gm, gn = -(-M // tm), -(-N // tn)
        assert gm * gn * THREADS[k] < 1 << 32, (M, N, K, NAMES[k])
        if k < 3:                                  # a grid of two dimensions
            assert gm <= 65535
