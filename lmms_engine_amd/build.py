"""Builds lmms_engine_amd/libmuon_hip.so from csrc/ with hipcc for gfx950, and the host-side Python module _scan beside it.

Run as `python -m lmms_engine_amd.build` or call build_library().  The library is built
in-tree, next to this file, so it travels with the source tree.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmuon_hip.so")
SOURCES = ["gemm_nt.hip", "elementwise.hip", "small_chain.hip", "multi_tensor.hip", "product.hip", "rows.hip", "api.hip"]
# Measurement kernels (MFMA-only loops) for the benchmark's operand-power legs: a library of their own, no part of the product.
PROBE_LIB = os.path.join(HERE, "libmuon_probe.so")
PROBE_SOURCES = ["probe.hip"]
# Reads lists of torch tensors for the optimizer step (host code; a Python module, since it handles Python objects).  Its name says
# which Python it is for, and it carries the version of the torch whose headers it was compiled with (checked when it is loaded).
SCAN_LIB = os.path.join(HERE, "_scan" + sysconfig.get_config_var("EXT_SUFFIX"))
# linear and gated_linear between torch and the library: host code too, under the same conditions, linked against the library beside it.
LAYERS_LIB = os.path.join(HERE, "_layers" + sysconfig.get_config_var("EXT_SUFFIX"))
# embedding, layer_norm, rms_norm and dropout, in the same way
ROWS_LIB = os.path.join(HERE, "_rows" + sysconfig.get_config_var("EXT_SUFFIX"))
# Packed-fp32 VALU forms stay off for every device function.
HIP_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-fPIC",
    "-std=c++17",
    "-fvisibility=hidden",  # the libraries export their extern "C" entry points and nothing else
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _compile_and_link(sources, lib, hipcc, verbose):
    objdir = os.path.join(CSRC, "build")
    os.makedirs(objdir, exist_ok=True)
    procs = []
    for src in sources:
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        cmd = [hipcc, *HIP_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs = []
    for src, obj, p in procs:
        out, _ = p.communicate()
        out = "\n".join(l for l in out.splitlines() if "not a recognized feature" not in l)
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed on {src}:\n{out}")
        if verbose and out.strip():
            print(out)
        objs.append(obj)
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", lib]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}")
    return lib


def _build_module(source, out, define, flags, verbose):
    """A Python module from one host source, with the headers of the torch that is installed."""
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths

    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-D{define}="{torch.__version__}"', *[f"-isystem{p}" for p in include_paths()], f"-isystem{sysconfig.get_paths()['include']}", os.path.join(CSRC, source), "-o", out,
           *[f"-L{p}" for p in library_paths()], *flags, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {source}:\n{r.stdout}")


def _build_scan(verbose):
    _build_module("scan.cpp", SCAN_LIB, "SCAN_TORCH_VERSION", [], verbose)


def _build_functions(source, out, define, hipcc, verbose):
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(hipcc)))
    flags = ["-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f"-isystem{os.path.join(rocm, 'include')}", f"-L{HERE}", "-l:" + os.path.basename(LIB),
             "-Wl,-rpath,$ORIGIN", "-lc10_hip"]
    _build_module(source, out, define, flags, verbose)


def built() -> bool:
    """Whether everything that the package loads is there."""
    return all(os.path.exists(p) for p in (LIB, SCAN_LIB, LAYERS_LIB, ROWS_LIB))


def build_library(verbose: bool = False) -> str:
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        raise RuntimeError("hipcc not found; cannot build libmuon_hip.so")
    _build_scan(verbose)
    _compile_and_link(PROBE_SOURCES, PROBE_LIB, hipcc, verbose)
    lib = _compile_and_link(SOURCES, LIB, hipcc, verbose)
    with ThreadPoolExecutor(2) as pool:  # torch's headers take half a minute each
        modules = [pool.submit(_build_functions, "layers.cpp", LAYERS_LIB, "LAYERS_TORCH_VERSION", hipcc, verbose),
                   pool.submit(_build_functions, "rows.cpp", ROWS_LIB, "ROWS_TORCH_VERSION", hipcc, verbose)]
        for m in modules:
            m.result()
    return lib


if __name__ == "__main__":
    print(build_library(verbose="-v" in sys.argv))
