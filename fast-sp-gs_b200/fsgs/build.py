"""Builds ``libfsgs.so`` (sm_100a) next to the sources.  ``python -m fsgs.build`` or ``fsgs.build.build()``."""
import importlib.util
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(PKG), "csrc")
LIB = os.path.join(os.path.dirname(PKG), "lib", "libfsgs.so")
HOST = os.path.join(os.path.dirname(PKG), "lib", "_fsgs_host.so")   # CPython extension over torch's headers
SOURCES = ["fsgs_preprocess.cu", "fsgs_bin.cu", "fsgs_blend.cu", "fsgs_knn.cu", "fsgs_epilogue.cu", "fsgs_loss.cu", "fsgs_compact.cu", "fsgs_step.cu", "fsgs_motion.cu",
           "fsgs_adamw.cu", "fsgs_balance.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "--expt-extended-lambda", "-Xcompiler", "-fPIC"]


def _has_torch():
    """Without torch (a host that uses the C ABI alone) the library is built and the host extension is not."""
    return importlib.util.find_spec("torch") is not None


def _stale():
    built = [LIB] + ([HOST] if _has_torch() else [])
    if not all(os.path.exists(f) for f in built):
        return True
    t = min(os.path.getmtime(f) for f in built)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(os.path.dirname(os.path.dirname(PKG)), "include", "fsgs.h"))
    return any(os.path.getmtime(d) > t for d in deps)


def _cuda_home():
    nvcc = shutil.which("nvcc")
    return os.path.dirname(os.path.dirname(os.path.realpath(nvcc))) if nvcc else "/usr/local/cuda"


def _host_command():
    """g++ command line of the host extension: torch's headers and libraries, this interpreter's headers."""
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    inc = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           sysconfig.get_paths()["include"], os.path.join(_cuda_home(), "include")]
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", os.path.join(CSRC, "fsgs_host.cpp"), "-o", HOST,
            "-Wl,--no-as-needed", "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"] + ["-I" + d for d in inc]


def build(force=False, verbose=False):
    """Compile every CUDA source for sm_100a and link the shared library, and, where torch is installed, compile the host
    extension beside it.  Returns the library path."""
    if not force and not _stale():
        return LIB
    os.makedirs(os.path.dirname(LIB), exist_ok=True)
    objs, procs = [], []
    for src in SOURCES:
        obj = os.path.join(os.path.dirname(LIB), src + ".o")
        cmd = ["nvcc", "-c", os.path.join(CSRC, src), "-o", obj] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else [])
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
        objs.append(obj)
    if _has_torch():
        cmd = _host_command()
        procs.append((cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for cmd, p in procs:
        out, _ = p.communicate()
        if verbose or p.returncode:
            sys.stderr.write(out)
        if p.returncode:
            raise RuntimeError("compilation failed: " + " ".join(cmd))
    subprocess.check_call(["nvcc", "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a",
                                                                  "-lcudart"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
