"""Compile the gfx950 HIP kernels and the C-ABI into liblbw_attn.so, and the block operators' binding to Python (host code
only) into _block.so, in-tree next to this file."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "liblbw_attn.so")
BLOCK = os.path.join(HERE, "_block.so")
SOURCES = ["lbw_abi.hip", "kv_requant.hip", "quant_q.hip", "prologue.hip", "cross_attn.hip", "fp8_quant.hip", "fp8_gemm.hip",
           "gated_norm.hip", "rotary.hip", "w4_gemm.hip", "attn_fwd.hip"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    # no packed-fp32 VALU ops anywhere
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc():
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return os.path.join(rocm, "bin", "hipcc")


def build_library(verbose=False):
    """Compile every HIP source into liblbw_attn.so (always recompiles). Returns the library path."""
    srcs = [os.path.join(HERE, "csrc", s) for s in SOURCES]
    tmp = LIB + ".tmp"
    cmd = [hipcc()] + HIPCC_FLAGS + ["-I", os.path.join(ROOT, "include")] + srcs + ["-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("hipcc failed building liblbw_attn.so")
    os.replace(tmp, LIB)
    return LIB


def build_binding(verbose=False):
    """Compile csrc/block_binding.cpp against this Python and torch (always recompiles; liblbw_attn.so has to be built).
    Returns the module's path."""
    import sysconfig
    from torch.utils import cpp_extension
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    tmp = BLOCK + ".tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch_cxx11_abi())}"]
    for d in (os.path.join(ROOT, "include"), sysconfig.get_paths()["include"], *cpp_extension.include_paths(),
              os.path.join(rocm, "include")):
        cmd += ["-isystem" if d != os.path.join(ROOT, "include") else "-I", d]
    cmd += [os.path.join(HERE, "csrc", "block_binding.cpp"), "-o", tmp, "-L", HERE, "-llbw_attn"]
    for d in cpp_extension.library_paths():
        cmd += ["-L", d]
    cmd += ["-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed building _block.so")
    os.replace(tmp, BLOCK)
    return BLOCK


def torch_cxx11_abi():
    import torch
    return torch._C._GLIBCXX_USE_CXX11_ABI


if __name__ == "__main__":
    print(build_library(verbose=True))
    print(build_binding(verbose=True))
