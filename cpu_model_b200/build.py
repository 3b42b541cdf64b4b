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


def newer(files, target):
    return not os.path.exists(target) or any(os.path.getmtime(f) > os.path.getmtime(target) for f in files)


def needs_build():
    csrc = [os.path.join(HERE, "csrc", f) for f in os.listdir(os.path.join(HERE, "csrc")) if f != "mxq_py.cpp"]
    return newer(csrc + [os.path.join(ROOT, "include", "mxq.h")], LIB)


def binding_tag(torch):
    """What a binding was built against: torch's C++ interface and Python's are their versions' own."""
    return "torch %s python %s" % (torch.__version__, sys.version.split()[0])


def binding_is_old(torch):
    if newer([os.path.join(HERE, "csrc", "mxq_py.cpp"), os.path.join(ROOT, "include", "mxq.h")], BINDING):
        return True
    try:
        with open(BINDING + ".tag") as f:
            return f.read() != binding_tag(torch)
    except OSError:
        return True


def build_binding(torch, verbose=False):
    """_serve.so: csrc/mxq_py.cpp against the installed torch and libmxq.so."""
    import sysconfig

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
    with open(BINDING + ".tag", "w") as f:
        f.write(binding_tag(torch))
    return BINDING


def build_library(verbose=False, ptxas_v=False):
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


def build(force=False, verbose=False, ptxas_v=False):
    """The library, which needs nvcc, and the binding, which needs torch with
    its headers: without them it is left out, and only its calls are missing."""
    if force or needs_build():
        build_library(verbose, ptxas_v)
    try:
        import torch
        from torch.utils import cpp_extension
        if not any(os.path.exists(os.path.join(i, "torch", "extension.h")) for i in cpp_extension.include_paths()):
            raise ImportError("torch has no headers")
    except (ImportError, OSError) as e:
        print("_serve.so (the serving calls' binding) is not built: %s" % e, file=sys.stderr)
        return LIB
    if force or binding_is_old(torch):
        build_binding(torch, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, ptxas_v="--ptxas-v" in sys.argv)
    print(LIB)
