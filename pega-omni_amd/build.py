"""Build libomni_attn.so for gfx950 in-tree with hipcc.

Usage: python pega-omni_amd/build.py   (or __graft_entry__.build()).
Every source under csrc/ is compiled to an object in _build/ and linked into
pega-omni_amd/libomni_attn.so, the library the C ABI in include/omni_attn.h
names. mirror/tensors.cpp (host code, against torch's headers) becomes
pega-omni_amd/omni_tensors.so, the Python mirror's checks of a call's tensors.
The library needs neither torch nor g++: it is linked whatever becomes of that
helper, which is left out where torch cannot be imported.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libomni_attn.so")
BUILD = os.path.join(HERE, "_build")
TENSORS = os.path.join(HERE, "omni_tensors.so")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wall",
    # Packed FP32 (v_pk_*_f32) stays off in every kernel.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


# Per-source additions. The decode kernels stream K/V and do little math:
# LLVM's memory-clause scheduling strategy groups their loads, 0.1-0.3% faster
# on every decode workload. The MFMA kernels were 1-3% slower under it.
SOURCE_FLAGS = {"decode.hip": ["-mllvm", "-amdgpu-sched-strategy=max-memory-clause"]}


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")))


def _compile(src: str) -> str:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    cmd = [HIPCC, *FLAGS, *SOURCE_FLAGS.get(os.path.basename(src), []), "-x", "hip", "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{r.stderr}")
    return obj


def _build_tensors() -> None:
    try:
        import torch
    except (ImportError, OSError) as e:
        print(f"{TENSORS} not built, torch cannot be imported ({e}): the C library does not need it, the Python "
              "mirror's 8-bit calls do", file=sys.stderr)
        return
    root = os.path.dirname(torch.__file__)
    inc, lib = os.path.join(root, "include"), os.path.join(root, "lib")
    tmp = TENSORS + ".tmp"
    built_for = "torch %s, Python %d.%d" % (torch.__version__, *sys.version_info[:2])
    cmd = ["g++", f'-DOMNI_BUILT_FOR="{built_for}"', "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           "-isystem", inc, "-isystem", os.path.join(inc, "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], os.path.join(HERE, "mirror", "tensors.cpp"), "-o", tmp,
           "-L" + lib, "-ltorch_python", "-ltorch_cpu", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on tensors.cpp:\n{r.stderr}")
    os.replace(tmp, TENSORS)


def build(verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    with ThreadPoolExecutor(max_workers=4) as ex:
        tensors = ex.submit(_build_tensors)
        objs = list(ex.map(_compile, sources()))
        tmp = OUT + ".tmp"
        cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
        os.replace(tmp, OUT)
        if verbose:
            print(f"built {OUT}")
        tensors.result()
    return OUT


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
