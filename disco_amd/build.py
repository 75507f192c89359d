"""Builds libdisco_hip.so (hand-written HIP kernels + C ABI) for gfx950 with hipcc.

The library is built IN-TREE (``disco_amd/csrc/libdisco_hip.so``) so that the binary travels with
the source tree; nothing is JIT-compiled at import time.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
ROOT = os.path.dirname(HERE)
SOURCES = ["disco_spmm.hip", "disco_stream.hip", "disco_schedule.hip", "disco_norm.hip", "disco_scorer.hip",
           "disco_build.hip", "disco_gather.hip", "disco_locality.hip",
           "disco_gradnorm.hip", "disco_residual.hip", "disco_residual_f32.hip", "disco_residual_f16.hip", "disco_residual_bf16.hip",
           "disco_residual_f32_f16.hip", "disco_residual_f32_bf16.hip"]
HEADERS = ["disco_internal.h", "disco_spmm_common.h", "disco_residual.h", os.path.join(ROOT, "include", "disco_hip.h")]
ARCH = "gfx950"


def lib_path(name: str = "libdisco_hip.so") -> str:
    return os.path.join(CSRC, name)


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


def _newest_source_mtime() -> float:
    paths = [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    paths += [h if os.path.isabs(h) else os.path.join(CSRC, h) for h in HEADERS]
    paths.append(os.path.abspath(__file__))
    return max(os.path.getmtime(p) for p in paths if os.path.exists(p))


def build_torch_lib(force: bool = False) -> str:
    """libdisco_torch.so: the torch operators of the residual join and the gradient norm, host code against torch's own headers
    and libraries."""
    out, src = lib_path("libdisco_torch.so"), os.path.join(CSRC, "disco_torch.cpp")
    needs = [src, os.path.join(ROOT, "include", "disco_hip.h"), os.path.abspath(__file__)]
    if not force and os.path.exists(out) and os.path.getmtime(out) >= max(map(os.path.getmtime, needs)):
        return out
    import torch
    from torch.utils.cpp_extension import include_paths, library_paths
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                           *("-I" + p for p in include_paths("cuda")), src, "-o", out, *("-L" + p for p in library_paths()), "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_hip"])
    return out


def build_lib(force: bool = False, extra_flags=(), name: str = "libdisco_hip.so", verbose: bool = False) -> str:
    out = lib_path(name)
    if not force and os.path.exists(out) and os.path.getmtime(out) >= _newest_source_mtime():
        return out
    hipcc = _hipcc()
    flags = ["-O3", "-std=c++17", "-fPIC", f"--offload-arch={ARCH}", "-fhip-fp32-correctly-rounded-divide-sqrt",
             "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-Wall", "-Wno-unused-function", f"-I{os.path.join(ROOT, 'include')}", f"-I{CSRC}"]
    # -packed-fp32-ops (the host pass warns that it does not know the feature): some forms of the packed float32
    # instructions that hipcc makes from ordinary float code have given wrong results on MI355X now and then
    flags += list(extra_flags)
    objdir = os.path.join(CSRC, "build", name.replace(".so", ""))
    os.makedirs(objdir, exist_ok=True)
    srcs = [s for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]

    def needs(src: str):
        heads = [h for h in HEADERS if h != "disco_residual.h" or src.startswith("disco_residual")]
        return [os.path.abspath(__file__), os.path.join(CSRC, src)] + [os.path.join(CSRC, h) for h in heads]

    def compile_one(src: str) -> str:
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        if not force and not extra_flags and os.path.exists(obj) and os.path.getmtime(obj) >= max(map(os.path.getmtime, needs(src))):
            return obj
        cmd = [hipcc, *flags, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.check_call(cmd)
        return obj

    with ThreadPoolExecutor(max_workers=min(6, len(srcs))) as ex:
        objs = list(ex.map(compile_one, srcs))
    cmd = [hipcc, "-shared", "-fPIC", f"--offload-arch={ARCH}", "-o", out, *objs]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.check_call(cmd)
    return out


def build_all(force: bool = False, verbose: bool = False) -> str:
    """The C library, then the torch operators beside it (which need g++ and torch's headers).  Returns the C library's path."""
    out = build_lib(force, verbose=verbose)
    build_torch_lib(force)
    return out


if __name__ == "__main__":
    print(build_all(force="--force" in sys.argv, verbose=True))
