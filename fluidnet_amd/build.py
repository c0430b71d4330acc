"""Build libfluidnet_hip.so in-tree with hipcc for gfx950 (cross-compiles without a GPU), and engine/_torch_ops.so, the host side of the
operators on torch tensors, with the host compiler against torch's headers.

    python -m fluidnet_amd.build [--force]

Both are git-ignored.
"""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libfluidnet_hip.so")
SOURCES = ["fnet_elementwise.hip", "fnet_loss.hip", "fnet_conv_ref.hip", "fnet_conv_mfma.hip", "fnet_optim.hip", "fnet_plan.hip", "fnet_rollout.hip",
           "fnet_block_norm.hip", "fnet_block_norm_f32.hip", "fnet_block_norm_bf16.hip", "fnet_block_norm_f16.hip",
           "fnet_tensor_list.hip"]
HEADERS = [os.path.join(CSRC, h) for h in ("fnet_common.h", "fnet_vec.h", "fnet_block_norm.h", "fnet_block_norm_fwd.h",
                                             "fnet_block_norm_bwd.h")] + [os.path.join(os.path.dirname(HERE), "include", "fluidnet_hip.h")]
# -packed-fp32-ops: hipcc makes v_pk_{add,mul,fma}_f32 of ordinary float code by itself, and some of their forms have given wrong results on
# MI355X now and then.  The scalar forms cost what little of the code arithmetic bounds (training step 35.7 -> 35.9 ms, rollout 5818 -> 5758
# scene-frames/s on one box).  (The host pass warns that it does not know the feature.)
FLAGS = ["--offload-arch=gfx950", "-O3", "-fPIC", "-std=c++17", "-ffp-contract=off", "-Wall", "-Wno-unused-function", "-Wno-unused-value",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

CXX = os.environ.get("CXX", "g++")
TORCH_OPS_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_OPS = os.path.join(HERE, "engine", "_torch_ops.so")


def _hipcc() -> str:
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    raise RuntimeError("hipcc not found")


def _stale(target: str, deps) -> bool:
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force: bool = False, verbose: bool = True) -> str:
    os.makedirs(LIBDIR, exist_ok=True)
    hipcc = _hipcc()
    objs = []
    jobs = []
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        obj = os.path.join(LIBDIR, s.replace(".hip", ".o"))
        objs.append(obj)
        if force or _stale(obj, [src, __file__] + HEADERS):      # the flags stand in this file
            jobs.append([hipcc, *FLAGS, "-c", src, "-o", obj])
    ops_obj = os.path.join(LIBDIR, "torch_ops.o")
    if force or _stale(ops_obj, [TORCH_OPS_SRC, __file__, HEADERS[-1]]):
        jobs.append([CXX, *_torch_flags(), "-c", TORCH_OPS_SRC, "-o", ops_obj])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"build failed:\n{' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        if verbose and r.stderr.strip():
            print(r.stderr, file=sys.stderr)

    with ThreadPoolExecutor(max_workers=min(6, max(1, len(jobs)))) as ex:
        list(ex.map(run, jobs))
    if force or jobs or _stale(LIB, objs):
        # -z defs: an unresolved kernel stub must fail the build here, not the dlopen on the GPU box
        run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-Wl,-z,defs", "-o", LIB, *objs])
    if force or jobs or _stale(TORCH_OPS, [ops_obj]):
        at = _torch_dir()
        run([CXX, "-shared", "-o", TORCH_OPS, ops_obj, f"-L{at}/lib", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip", "-lamdhip64"])
    return LIB


def _torch_dir() -> str:
    import torch
    return os.path.dirname(torch.__file__)


def _torch_flags():
    import sysconfig

    import torch
    at = _torch_dir()
    include = (f"{at}/include", f"{at}/include/torch/csrc/api/include", sysconfig.get_path("include"), os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include"))
    return ["-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-isystem{i}" for i in include)]


if __name__ == "__main__":
    print(build(force="--force" in sys.argv))
