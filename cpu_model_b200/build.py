"""Build recipe for libmxq.so (sm_100a) and _serve.so, in-tree next to this file.

    python -m cpu_model_b200.build

nvcc compiles the CUDA sources for sm_100a only and links a shared library
with a plain C-ABI (include/mxq.h); no torch headers are involved.  _serve.so is
the Python binding of its serving calls (csrc/mxq_py.cpp), host code over torch's
tensors, linked to the library beside it.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SOURCES = ["mxq_api.cu", "mxq_quant.cu", "mxq_gemv.cu", "mxq_rgemv.cu", "mxq_bgemv.cu", "mxq_gemm.cu", "mxq_moe.cu",
           "mxq_ops.cu", "mxq_decoder_kernels.cu", "mxq_decoder.cu", "mxq_cogemv.cu",
           "mxq_tp.cu", "mxq_kv.cu", "mxq_kvattn.cu", "mxq_kvprompt.cu", "mxq_logprob.cu"]
LIB = os.path.join(HERE, "libmxq.so")
BINDING = os.path.join(HERE, "_serve.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    "-I" + os.path.join(ROOT, "include"),
]


def needs_build():
    if not os.path.exists(LIB) or not os.path.exists(BINDING):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(BINDING))
    deps = [os.path.join(HERE, "csrc", f) for f in os.listdir(os.path.join(HERE, "csrc"))]
    deps.append(os.path.join(ROOT, "include", "mxq.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def build_binding(verbose=False):
    """_serve.so: csrc/mxq_py.cpp against the installed torch and libmxq.so."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ext
    inc = ext.include_paths() + [sysconfig.get_paths()["include"], "/usr/local/cuda/include", os.path.join(ROOT, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_serve",
           "-DTORCH_API_INCLUDE_EXTENSION_H", "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI]
    cmd += ["-isystem" + i for i in inc] + [os.path.join(HERE, "csrc", "mxq_py.cpp"), "-o", BINDING + ".tmp"]
    cmd += ["-L" + p for p in ext.library_paths()] + ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    cmd += ["-L" + HERE, "-l:libmxq.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd))
    subprocess.check_call(cmd)
    os.replace(BINDING + ".tmp", BINDING)
    return BINDING


def build(force=False, verbose=False, ptxas_v=False):
    if not force and not needs_build():
        return LIB
    objs = []
    for src in SOURCES:
        obj = os.path.join(HERE, "csrc", src.replace(".cu", ".o"))
        cmd = [NVCC] + FLAGS + (["-Xptxas", "-v"] if ptxas_v else []) + [
            "-c", os.path.join(HERE, "csrc", src), "-o", obj]
        if verbose:
            print(" ".join(cmd))
        subprocess.check_call(cmd)
        objs.append(obj)
    tmp = LIB + ".tmp"
    subprocess.check_call([NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a",
                           "-o", tmp] + objs)
    os.replace(tmp, LIB)
    for o in objs:
        os.remove(o)
    build_binding(verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_v="--ptxas-v" in sys.argv)
    print(LIB)
