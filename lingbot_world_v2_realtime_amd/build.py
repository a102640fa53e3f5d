"""Compile the gfx950 HIP kernels and the C-ABI into liblbw_attn.so, and the block operators' binding to Python (host code
only) into _block.so, in-tree next to this file."""
import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "liblbw_attn.so")
BLOCK = os.path.join(HERE, "_block.so")
SOURCES = ["lbw_abi.hip", "kv_requant.hip", "quant_q.hip", "prologue.hip", "cross_attn.hip", "fp8_quant.hip", "fp8_gemm.hip",
           "gated_norm.hip", "rotary.hip", "w4_gemm.hip", "norm_rotary.hip", "packed_attn.hip", "packed_attn_bwd.hip", "kv4.hip",
           "attn_fwd.hip"]
BINDING = ["block_binding.cpp", "causal_binding.cpp"]

HIPCC_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
    # no packed-fp32 VALU ops anywhere
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc():
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return os.path.join(rocm, "bin", "hipcc")


def jobs():
    """Compilers side by side: MAX_JOBS where it is a number, else 8; no more than processors or sources."""
    want = os.environ.get("MAX_JOBS", "")
    return max(1, min(int(want) if want.isdecimal() else 8, os.cpu_count() or 1, len(SOURCES)))


def build_library(verbose=False):
    """Compile every HIP source, several side by side, and link them into liblbw_attn.so (always recompiles). Returns the library
    path."""
    tmp = LIB + ".tmp"

    def run(args):
        cmd = [hipcc()] + HIPCC_FLAGS + args
        if verbose:
            print(" ".join(cmd), flush=True)
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("hipcc failed building liblbw_attn.so")

    with tempfile.TemporaryDirectory() as objects, ThreadPoolExecutor(jobs()) as pool:
        outs = [os.path.join(objects, s + ".o") for s in SOURCES]
        list(pool.map(run, [["-I", os.path.join(ROOT, "include"), "-c", os.path.join(HERE, "csrc", s), "-o", o]
                            for s, o in zip(SOURCES, outs)]))
        run(["-shared", *outs, "-o", tmp])
    os.replace(tmp, LIB)
    return LIB


def build_binding(verbose=False):
    """Compile the bindings (csrc/*_binding.cpp) against this Python and torch (always recompiles; liblbw_attn.so has to be built).
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
    cmd += [os.path.join(HERE, "csrc", s) for s in BINDING] + ["-o", tmp, "-L", HERE, "-llbw_attn"]
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
