"""Build the sm_100a shared library in-tree with nvcc (no GPU needed to compile)."""
from __future__ import annotations

import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmegaattn_b200.so")
# Same sources with -DMA_AUDIT: the scheduler counts every finished unit of work (tests
# assert exactly-once execution with it).  Kept out of the product build because even a
# never-taken branch in the scheduler role shifts the attention loop's code generation
# (measured: +1.2 % on the attention stage).
LIB_AUDIT = os.path.join(HERE, "libmegaattn_b200_audit.so")
SOURCES = ["fused_prefill.cu", "cabi.cu", "noalloc.cu", "residual_rmsnorm.cu", "rope.cu",
           "detile.cu", "meta_upload.cu", "step.cu", "meta.cpp", "rmsnorm_quant.cu", "linear_quant.cu", "rope_append.cu",
           "dequant.cu"]
HEADERS = ["ptx.cuh", "kparams.h", "launch.cuh", "paged.cuh", "append_place.h", "linear_form.h",
           os.path.join("..", "..", "include", "megaattn_b200.h")]


def torch_version() -> str:
    """Of the torch that is installed, read without importing it where it stands in the usual place."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return "none"
    try:
        with open(os.path.join(os.path.dirname(spec.origin), "version.py")) as f:
            found = re.search(r"^__version__\b[^=\n]*= *['\"]([^'\"]+)", f.read(), re.M)
    except (OSError, TypeError):
        found = None
    if found:
        return found.group(1)
    import torch
    return str(torch.__version__)


# The operators' calls natively (csrc/calls.cpp): a Python module over torch's tensors, which hands the C ABI's
# entry points plain pointers.  Host code only.  It works with the torch it was built for, whose version is part of
# the name: behind another torch it is missing, and built again.
LIB_CALLS = os.path.join(HERE, f"_calls_torch{torch_version()}" + sysconfig.get_config_var("EXT_SUFFIX"))
CALLS = ["calls.cpp", os.path.join("..", "..", "include", "megaattn_b200.h")]


def _stale(lib: str = None) -> bool:
    lib = lib or LIB
    if not os.path.exists(lib):
        return True
    t = os.path.getmtime(lib)
    return any(os.path.getmtime(os.path.join(CSRC, f)) > t for f in (CALLS if lib == LIB_CALLS else SOURCES + HEADERS))


def build(force: bool = False, verbose: bool = False, audit: bool = False) -> str:
    """Compile ``csrc/*.cu`` into ``libmegaattn_b200.so`` (or, with ``audit``, into
    ``libmegaattn_b200_audit.so``) next to this file."""
    LIB = LIB_AUDIT if audit else globals()["LIB"]
    nvcc = os.environ.get("NVCC", "nvcc")
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3",
           "-std=c++17", "-Xcompiler", "-fPIC", "-shared"]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    if audit:
        cmd += ["-DMA_AUDIT"]
    return _compile(LIB, cmd + [os.path.join(CSRC, f) for f in SOURCES], force, verbose)


def _cuda_include() -> str:
    """Where CUDA's headers are: of CUDA_HOME, or of the nvcc that compiles the kernels."""
    nvcc = shutil.which(os.environ.get("NVCC", "nvcc"))
    home = os.environ.get("CUDA_HOME") or (os.path.dirname(os.path.dirname(os.path.realpath(nvcc))) if nvcc else "/usr/local/cuda")
    return os.path.join(home, "include")


def build_calls(force: bool = False) -> str:
    """Compile ``csrc/calls.cpp`` against the torch that is installed."""
    import torch
    at = os.path.dirname(torch.__file__)
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f'-DMA_TORCH_VERSION="{torch.__version__}"', "-I" + sysconfig.get_paths()["include"],
           "-I" + _cuda_include(), "-I" + os.path.join(at, "include"),
           "-I" + os.path.join(at, "include", "torch", "csrc", "api", "include"), os.path.join(CSRC, "calls.cpp"),
           "-L" + os.path.join(at, "lib"), "-Wl,-rpath," + os.path.join(at, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_cuda", "-ltorch_python"]
    return _compile(LIB_CALLS, cmd, force)


def _compile(LIB: str, cmd: list, force: bool, verbose: bool = False) -> str:
    if not force and not _stale(LIB):
        return LIB
    # Several processes (one per GPU under torchrun) may get here at once: one builds, into a
    # temporary file that is renamed over the library in one step, the others wait on the
    # lock and find the library fresh.
    import fcntl
    with open(LIB + ".lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        if not force and not _stale(LIB):
            return LIB
        tmp = f"{LIB}.{os.getpid()}.tmp"
        res = subprocess.run(cmd + ["-o", tmp], capture_output=True, text=True)
        if res.returncode != 0:
            if os.path.exists(tmp):
                os.remove(tmp)
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed:\n" + res.stdout + res.stderr)
        os.replace(tmp, LIB)
        if verbose:
            sys.stderr.write(res.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build(force=True, audit=True))
    print(build_calls(force=True))
