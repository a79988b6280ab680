"""Builds the gfx950 encoder library libud_encoder.so in-tree with hipcc.

    python universal-dictator_amd/build.py

Objects go to universal-dictator_amd/_build/, the library to universal-dictator_amd/lib/.
Every HIP source is compiled for gfx950 only.
"""
import concurrent.futures
import os
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
SRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(PKG, "_build")
LIB_DIR = os.path.join(PKG, "lib")
LIB = os.path.join(LIB_DIR, "libud_encoder.so")
SOURCES = ["attention.hip", "attention_dense.hip", "gemm.hip", "norm_conv.hip", "encoder.hip", "runtime.hip", "decode.hip", "cache.hip", "window.hip", "prefill.hip", "subsample.hip", "rnnt.hip", "mel.hip", "peaks.hip", "safetensors.cpp", "streamer.cpp", "tokenizer.cpp"]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden",
    # no packed-fp32 VALU instructions in device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


# Per-file flags.  attention_dense.hip: the machine scheduler's max-ilp strategy (the offline
# attention kernel is latency-bound at two waves per SIMD; measured 148.1-148.4 -> 144.9-145.2 us
# per launch at 8 x 1500 frames, bit-identical output).
FILE_FLAGS = {"attention_dense.hip": ["-mllvm", "-amdgpu-sched-strategy=max-ilp"]}


def _run(cmd):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in r.stdout.splitlines() if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError("command failed (%d): %s\n%s" % (r.returncode, " ".join(cmd), out))
    return out


def build(verbose=False):
    os.makedirs(OBJ, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)

    def compile_one(src):
        obj = os.path.join(OBJ, src.rsplit(".", 1)[0] + ".o")
        _run([HIPCC] + FLAGS + FILE_FLAGS.get(src, []) + ["-c", os.path.join(SRC, src), "-o", obj])
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    tmp = LIB + ".tmp"
    _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp] + objs)
    os.replace(tmp, LIB)
    if verbose:
        print("built", LIB)
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
