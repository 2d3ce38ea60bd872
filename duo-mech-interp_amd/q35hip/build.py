"""Build recipe of libq35hip.so: every csrc/*.hip compiled for gfx950 with hipcc, linked into one shared library that
exports the C ABI declared in include/q35hip.h; and of the Python extension _paged_host.so (csrc/paged_host.cpp, host code over
torch's C++ interface). Both land next to this file (in-tree) so that they travel with the source tree and are what the
Python package loads.

    python -m q35hip.build          (from duo-mech-interp_amd/)
"""
import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)                      # duo-mech-interp_amd/
REPO = os.path.dirname(ROOT)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD_DIR = os.path.join(ROOT, "_build")
LIB_NAME = "libq35hip.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
HOST_PATH = os.path.join(PKG_DIR, "_paged_host.so")

ARCH = "gfx950"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CXXFLAGS = [
    f"--offload-arch={ARCH}", "-O3", "-std=c++17", "-fPIC", "-I" + INCLUDE, "-I" + CSRC,
    # packed fp32 VALU ops are kept out of the generated code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".hip"))


def _compile(src):
    obj = os.path.join(BUILD_DIR, os.path.basename(src)[:-4] + ".o")
    cmd = [HIPCC] + CXXFLAGS + ["-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(line for line in (r.stderr or "").splitlines() if noise not in line)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src}:\n{err}")
    return obj


def _build_host():
    """HOST_PATH: no device code, torch's libraries (loaded before it) by name."""
    import torch
    t = os.path.dirname(torch.__file__)
    tmp = HOST_PATH + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I" + INCLUDE,
           "-I" + os.path.join(t, "include"), "-I" + os.path.join(t, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], os.path.join(CSRC, "paged_host.cpp"), "-o", tmp,
           "-L" + os.path.join(t, "lib"), "-lc10", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"paged_host.cpp failed:\n{r.stderr}")
    os.replace(tmp, HOST_PATH)


def build(verbose=False, jobs=None):
    """Compile every kernel source and link LIB_PATH, and HOST_PATH beside it. Always rebuilds. The C library needs hipcc
    alone: where the extension cannot be built (no g++, no Python headers) a warning says why, and the ops that need it raise."""
    if not os.path.exists(HIPCC):
        raise RuntimeError(f"hipcc not found at {HIPCC}")
    os.makedirs(BUILD_DIR, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(len(srcs), max(1, (os.cpu_count() or 4)))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as ex:
        host = ex.submit(_build_host)
        objs = list(ex.map(_compile, srcs))
    tmp = LIB_PATH + ".tmp"
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp] + objs
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB_PATH)
    failed = host.exception()
    if failed is not None:
        if os.path.exists(HOST_PATH):
            os.remove(HOST_PATH)  # (an earlier one's calls need not fit this library)
        warnings.warn(f"q35hip: {HOST_PATH} could not be built, the paged-cache ops will raise: {failed}")
    if verbose:
        print(f"built {LIB_PATH} from {len(srcs)} sources" + ("" if failed is not None else f", and {HOST_PATH}"))
    return LIB_PATH


def clean():
    shutil.rmtree(BUILD_DIR, ignore_errors=True)


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
