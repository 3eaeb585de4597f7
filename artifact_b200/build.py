"""In-tree build of the native libraries.

* ``_lib/librof_b200.so`` — CUDA kernels + plan builder + the C ABI declared in
  ``include/rof_b200.h``; compiled by nvcc for sm_100a only.
* ``_lib/librof_host.so`` — host-only helpers (synthetic graph generators, the
  reuse-group search); compiled by g++ with OpenMP.
* ``_lib/rof_torch.so`` — autograd nodes of layer norm and dropout over the C ABI
  (``csrc/torch``); compiled by g++ against the installed torch.

The first two are plain shared objects loaded with ctypes and know nothing of torch; the third is a
Python module that links against the first and against torch.
Run ``python -m artifact_b200.build`` (or ``__graft_entry__.build()``).
"""
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "_lib")
INCLUDE = os.path.join(ROOT, "include")

CUDA_SOURCES = ["plan.cu", "kernels.cu", "api.cu", "stages.cu", "static_scratch.cu", "norm.cu",
                "norm_f32.cu", "norm_bf16.cu", "norm_f16.cu",
                "norm_tile_f32.cu", "norm_tile_bf16.cu", "norm_tile_f16.cu"]
HOST_SOURCES = [os.path.join("host", "graphgen.cpp"), os.path.join("host", "reuse_search.cpp")]

NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-Xcompiler", "-fPIC,-fopenmp,-O3",
    "--expt-relaxed-constexpr",
    # no implicit contraction: the kernels round where the source says so.  The GCN terms use an
    # explicit fused multiply-add (one rounding where upstream's __fmul_rn + add has two,
    # reuse_conv_kernel.cu:270); scales, epilogue and the pre-scaling pass are separate roundings
    "-fmad=false",
]


def _nvcc():
    return shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps if os.path.exists(d))


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)


def cuda_lib_path():
    return os.path.join(LIB, "librof_b200.so")


def host_lib_path():
    return os.path.join(LIB, "librof_host.so")


def torch_lib_path():
    return os.path.join(LIB, "rof_torch.so")


def build_cuda(force=False, verbose=True, ptxas_info=False):
    os.makedirs(LIB, exist_ok=True)
    srcs = [os.path.join(CSRC, s) for s in CUDA_SOURCES if os.path.exists(os.path.join(CSRC, s))]
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hdrs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    target = cuda_lib_path()
    if not force and not _stale(target, srcs + hdrs + [os.path.abspath(__file__)]):
        return target
    cmd = [_nvcc(), "--threads", "0"] + NVCC_FLAGS + ["-I", INCLUDE, "-I", CSRC, "-shared", "-o", target] + srcs
    if ptxas_info:
        cmd += ["-Xptxas", "-v"]
    cmd += ["-lcudart", "-lgomp"]
    _run(cmd, verbose)
    return target


def build_host(force=False, verbose=True):
    os.makedirs(LIB, exist_ok=True)
    srcs = [os.path.join(CSRC, s) for s in HOST_SOURCES if os.path.exists(os.path.join(CSRC, s))]
    target = host_lib_path()
    if not force and not _stale(target, srcs + [os.path.abspath(__file__)]):
        return target
    cmd = ["g++", "-O3", "-std=c++17", "-fPIC", "-shared", "-fopenmp", "-march=x86-64-v2",
           "-o", target] + srcs
    _run(cmd, verbose)
    return target


def torch_root():
    """the installed torch's folder, where it has its C++ headers; else None (nothing is imported)"""
    spec = importlib.util.find_spec("torch")
    root = os.path.dirname(spec.origin) if spec is not None and spec.origin else None
    return root if root and os.path.exists(os.path.join(root, "include", "torch", "csrc", "autograd", "custom_function.h")) else None


def _torch_stamp():
    """which torch rof_torch.so is built against: its folder and version"""
    root = torch_root()
    if root is None:
        raise RuntimeError("rof_torch.so needs an installed torch with its C++ headers")
    with open(os.path.join(root, "version.py")) as f:
        return root + "\n" + f.read()


def build_torch(force=False, verbose=True):
    cuda = build_cuda(verbose=verbose)
    src = os.path.join(CSRC, "torch", "norm_torch.cpp")
    target, stamp = torch_lib_path(), os.path.join(LIB, "rof_torch.stamp")
    against = _torch_stamp()
    same = os.path.exists(stamp) and open(stamp).read() == against
    if not force and same and not _stale(target, [src, os.path.join(INCLUDE, "rof_b200.h"), os.path.abspath(__file__)]):
        return target
    import torch
    root = os.path.dirname(os.path.abspath(torch.__file__))
    cuda_home = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI), "-I", INCLUDE]
    for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
              os.path.join(cuda_home, "include"), sysconfig.get_paths()["include"]):
        cmd += ["-isystem", d]
    cmd += [src, "-o", target, "-L" + LIB, "-l:" + os.path.basename(cuda), "-Wl,-rpath,$ORIGIN", "-L" + os.path.join(root, "lib"),
            "-Wl,-rpath," + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"]
    _run(cmd, verbose)
    with open(stamp, "w") as f:
        f.write(against)
    return target


def build_all(force=False, verbose=True):
    """-> the CUDA library and the host library (rof_torch.so is built beside them, where torch and its headers are installed)"""
    libs = build_cuda(force, verbose), build_host(force, verbose)
    if torch_root() is not None:
        build_torch(force, verbose)
    else:
        print("rof_torch.so is not built: torch with its C++ headers is not installed (artifact_b200.norm needs it; the C ABI does not)",
              file=sys.stderr, flush=True)
    return libs


if __name__ == "__main__":
    build_all(force="--force" in sys.argv, verbose=True)
