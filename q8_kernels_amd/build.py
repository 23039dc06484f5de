"""Builds libq8_hip.so (gfx950) from q8_kernels_amd/csrc/*.hip with hipcc, and _torch_ops.so (host code: tensor checks and
autograd of the operators whose host cost counts) from csrc/torch_ops.cpp against the installed torch.

Usage:  python -m q8_kernels_amd.build        (always recompiles)
The shared libraries are written next to this file; nothing is installed.
"""
import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libq8_hip.so")
OPS = os.path.join(HERE, "_torch_ops.so")
SOURCES = ["api.hip", "rows.hip", "fused.hip", "elementwise.hip", "gemm.hip", "attn.hip", "layernorm.hip", "rotary.hip", "cross_attn.hip",
           "cross_attn_bwd.hip"]
# packed fp32 VALU forms are disabled on purpose (they have miscomputed on this hardware pool)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc():
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "hipcc"


def _compile(src):
    obj = os.path.join(HERE, "build", os.path.splitext(src)[0] + ".o")
    cmd = [_hipcc(), *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    err = "\n".join(l for l in r.stderr.splitlines() if "is not a recognized feature" not in l)
    if r.returncode != 0:
        raise RuntimeError("hipcc failed for %s:\n%s" % (src, err))
    return obj, err


def _compile_ops():
    """csrc/torch_ops.cpp -> build/torch_ops.o; the flags that make it link with torch."""
    import sysconfig

    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    obj = os.path.join(HERE, "build", "torch_ops.o")
    includes = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), "/opt/rocm/include",
                sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_torch_ops",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    cmd += [a for i in includes for a in ("-isystem", i)] + ["-c", os.path.join(CSRC, "torch_ops.cpp"), "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for torch_ops.cpp:\n" + r.stderr)
    return [obj, "-L" + os.path.join(root, "lib"), "-L" + HERE, "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"]


def build(verbose=True):
    os.makedirs(os.path.join(HERE, "build"), exist_ok=True)
    with concurrent.futures.ThreadPoolExecutor(max_workers=5) as ex:
        ops = ex.submit(_compile_ops)
        results = list(ex.map(_compile, SOURCES))
        ops_link = ops.result()
    objs = [o for o, _ in results]
    if verbose:
        for (_, err), src in zip(results, SOURCES):
            if err.strip():
                print("[%s]\n%s" % (src, err), file=sys.stderr)
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stderr)
    r = subprocess.run(["g++", "-shared", "-o", OPS, *ops_link, "-l:" + os.path.basename(LIB), "-Wl,-rpath,$ORIGIN"], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("link failed:\n" + r.stderr)
    if verbose:
        print("built", LIB)
        print("built", OPS)
    return LIB


if __name__ == "__main__":
    build()
