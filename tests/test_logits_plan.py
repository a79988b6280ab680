"""CPU checks of ud_logits_process's split of a vocabulary (csrc/logits.hip, its host function compiled with the host compiler): the
workspace holds a key for each segment, and never shrinks as a batch or a vocabulary grows."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import test_gpu_long_lists as long_lists
from conftest import ROOT


@pytest.fixture(scope="module")
def segment(tmp_path_factory):
    """Tokens of a segment for (n, vocab)."""
    text = open(os.path.join(ROOT, "universal-dictator_amd", "csrc", "logits.hip")).read()
    fn = re.search(r"static int logit_segment\(.*?\n\}\n", text, re.S).group(0)
    d = tmp_path_factory.mktemp("logits")
    (d / "s.cpp").write_text('#include <cstdint>\n%s\nextern "C" int pick(long long n, long long vocab) { return logit_segment(n, vocab); }\n' % fn)
    so = str(d / "s.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(d / "s.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    lib.pick.argtypes = [ctypes.c_longlong] * 2
    return lib.pick


VOCABS = [1, 100, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32001, 32768, 32769, 65537, 131072, 131073, 200000, 1 << 20, 1 << 24]


def test_a_workspace_serves_smaller_batches(ud):
    sizes = np.array([[ud.logits_workspace_bytes(n, v) for v in VOCABS] for n in [*range(1, 301), 511, 512, 513, 4096, 65535]])
    assert np.all(np.diff(sizes, axis=0) >= 0) and np.all(np.diff(sizes, axis=1) >= 0)


def test_a_workspace_holds_every_segment(ud, segment):
    rng = np.random.default_rng(1)
    sizes = [(n, v) for n in [*range(1, 301), 511, 512, 513, 65535] for v in VOCABS]
    sizes += [tuple(int(x) for x in np.exp(rng.uniform(0, [11.09, 16.63]))) for _ in range(20000)]
    for n, v in sizes:
        need = 8 * n * -(-v // segment(n, v))
        assert need <= ud.logits_workspace_bytes(n, v) <= max(need, 8 * 512) or segment(n, v) == 2048, (n, v)


def test_long_lists_reach_every_segment(segment):
    """The GPU tests of long lists take the segments that they say, each size of them."""
    for n, v, tokens in long_lists.SIZES:
        assert segment(n, v) == tokens, (n, v)
    assert {s for _, _, s in long_lists.SIZES} == {2048, 4096, 8192, 16384, 32768}
