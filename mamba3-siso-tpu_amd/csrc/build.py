"""Compile the gfx950 HIP kernels and the C ABI into csrc/libm3s.so, and the autograd nodes in C++
into csrc/m3s_nodes.so (in-tree).

    python mamba3-siso-tpu_amd/csrc/build.py [--jobs N]

Every source is rebuilt on each call. Flags: gfx950 only; packed-FP32 ops disabled
(the compiler must not emit v_pk_{add,mul,fma}_f32). The nodes are host code, built against the
headers of the installed torch.
"""

from __future__ import annotations

import argparse
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCES = ["m3s_abi.hip", "m3s_fwd.hip", "m3s_bwd.hip", "m3s_decode.hip", "m3s_prep.hip",
           "m3s_norm.hip", "m3s_layout.hip", "m3s_mlp.hip",
           "m3s_rms.hip", "m3s_optim.hip", "m3s_wgrad.hip", "m3s_gemv.hip", "m3s_embed.hip",
           "m3s_vocab.hip"]
LIB = os.path.join(HERE, "libm3s.so")
NODES = os.path.join(HERE, "m3s_nodes.so")
BUILD_DIR = os.path.join(HERE, "_build")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall",
    "-Wno-unused-function",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]


def compile_one(src: str) -> str:
    obj = os.path.join(BUILD_DIR, src.replace(".hip", ".o"))
    cmd = [HIPCC, *FLAGS, "-c", os.path.join(HERE, src), "-o", obj]
    res = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(ln for ln in res.stderr.splitlines() if noise not in ln)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    if err.strip():
        print(err, file=sys.stderr)
    return obj


def build_nodes() -> None:
    """The node module: host code by the C++ compiler, its symbols from the torch that imports it."""
    torch = importlib.util.find_spec("torch").submodule_search_locations[0]
    includes = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"),
                sysconfig.get_paths()["include"], os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")]
    tmp = NODES + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
           "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", *[f for i in includes for f in ("-isystem", i)],
           os.path.join(HERE, "m3s_nodes.cpp"), "-o", tmp, "-L" + os.path.join(torch, "lib"),
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10_hip", "-lc10"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"building m3s_nodes failed:\n{res.stderr}")
    if res.stderr.strip():
        print(res.stderr, file=sys.stderr)
    os.replace(tmp, NODES)


def main(argv=None) -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=min(8, os.cpu_count() or 1))
    args = ap.parse_args(argv)
    os.makedirs(BUILD_DIR, exist_ok=True)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(HERE, s))]
    with ThreadPoolExecutor(args.jobs) as ex:
        nodes = ex.submit(build_nodes)
        objs = list(ex.map(compile_one, srcs))
        nodes.result()
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", tmp]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)
    print(f"built {LIB} and {NODES}")


if __name__ == "__main__":
    main()
