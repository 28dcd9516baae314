"""Compile libdynamis_graph.so (gfx950) in-tree with hipcc, and _torch_layer.so, which calls it from torch.

The library needs no torch: it is linked first, whatever becomes of _torch_layer.so.  Where there is no torch at
all it is all that is built.

    python -m dynamis_amd.build            # or dynamis_amd.build.build()

Flags: -ffp-contract=off keeps the canonical fp64 predicate's operation order exactly
as written (explicit fma only); packed fp32 ops are disabled for the target.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libdynamis_graph.so")
TORCH_LAYER = os.path.join(HERE, "_torch_layer.so")
SOURCES = ["dg_graph.hip", "dg_sfc.hip", "dg_halo.hip", "dg_batch.hip", "dg_neighbors.hip",
           "dg_attention.hip", "dg_attention_mfma.hip", "dg_grouped.hip", "dg_rotate.hip",
           "dg_route.hip", "dg_exchange.hip"]
ARCH = os.environ.get("DG_OFFLOAD_ARCH", "gfx950")

ROCM = "/opt/rocm"
HIPCC = os.environ.get("HIPCC", os.path.join(ROCM, "bin", "hipcc"))
CXX = os.environ.get("CXX", "g++")
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-I" + os.path.join(ROOT, "include"),
    "-Wall",
    "-Wextra",
]


def _run(cmd):
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(l for l in r.stdout.splitlines() if "packed-fp32-ops" not in l)
    if r.returncode != 0:
        raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + " ".join(cmd) + "\n" + out)
    return out


def _torch_layer() -> str:
    """The operators' calls from torch (host code alone): a module of the interpreter, on torch's C++ interface."""
    import sysconfig

    try:
        import torch
    except ImportError:
        return "no torch: _torch_layer.so is not built"
    from torch.utils import cpp_extension

    tmp = TORCH_LAYER + ".tmp"
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    out = _run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-DUSE_ROCM=1", "-D__HIP_PLATFORM_AMD__=1",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
                *("-isystem" + p for p in (*cpp_extension.include_paths(), os.path.join(ROCM, "include"),
                                           sysconfig.get_paths()["include"])),
                os.path.join(CSRC, "torch_layer.cpp"), "-o", tmp, "-L" + libs, "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch",
                "-ltorch_python"])
    os.replace(tmp, TORCH_LAYER)
    return out


def build(verbose: bool = False) -> str:
    bdir = os.path.join(HERE, "_build")
    os.makedirs(bdir, exist_ok=True)
    objs = [os.path.join(bdir, src.replace(".hip", ".o")) for src in SOURCES]
    with ThreadPoolExecutor(4) as pool:
        layer = pool.submit(_torch_layer)
        jobs = [pool.submit(_run, [HIPCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]) for src, obj in zip(SOURCES, objs)]
        out = [job.result() for job in jobs]
        tmp = LIB + ".tmp"
        out.append(_run([HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs]))
        os.replace(tmp, LIB)
        out.append(layer.result())
    if verbose:
        print(*(text for text in out if text.strip()), sep="\n")
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
