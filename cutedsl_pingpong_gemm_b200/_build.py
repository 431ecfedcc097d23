"""Build recipe for the sm_100a shared library (``libcpgemm.so``), built in-tree.

The library holds the C ABI of ``include/cpgemm.h`` in three translation units, compiled side
by side: ``csrc/capi.cu`` (the tcgen05 GEMM kernels, the FP8 quantiser and the scheduler/FastDivmod
device helpers), ``csrc/capi_moe.cu`` (the INT8 quantiser and the operators around the experts'
products) and ``csrc/capi_attention.cu`` (norm and rotation of heads, linear attention).  It links
the CUDA runtime statically and reaches ``cuTensorMapEncodeTiled`` through the runtime's driver entry-point
query, so it needs no link against ``libcuda``.
"""
import os
import shutil
import subprocess
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_NAME = "libcpgemm.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)

SOURCES = [os.path.join(CSRC, f) for f in ("capi.cu", "capi_moe.cu", "capi_attention.cu")]
# Every source and header of csrc/ and the public header: a change to any of them rebuilds.
DEPENDS = SOURCES + sorted(
    os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))
) + [os.path.join(INCLUDE, "cpgemm.h")]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "--expt-relaxed-constexpr",
]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def needs_build() -> bool:
    if not os.path.exists(LIB_PATH):
        return True
    t = os.path.getmtime(LIB_PATH)
    return any(os.path.getmtime(s) > t for s in DEPENDS if os.path.exists(s))


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile ``libcpgemm.so`` next to this file (skipped when it is newer than its sources)."""
    if not force and not needs_build():
        return LIB_PATH
    tmp = LIB_PATH + ".tmp"
    nvcc = [nvcc_path(), *NVCC_FLAGS]
    with tempfile.TemporaryDirectory() as work:
        objects = [os.path.join(work, os.path.basename(s) + ".o") for s in SOURCES]
        compiles = [[*nvcc, f"-I{INCLUDE}", f"-I{CSRC}", "-c", s, "-o", o]
                    for s, o in zip(SOURCES, objects)]
        running = [_start(cmd, verbose) for cmd in compiles]
        # Every compiler ends before the first failure is raised (and its folder goes).
        results = [(p, *p.communicate()) for p in running]
        for p, out, err in results:
            _check(p, out, err)
        p = _start([*nvcc, "-shared", *objects, "-o", tmp], verbose)
        _check(p, *p.communicate())
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def _start(cmd, verbose):
    if verbose:
        print(" ".join(cmd))
    return subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)


def _check(p, out, err):
    if p.returncode != 0:
        raise RuntimeError(f"nvcc failed ({p.returncode}):\n{out}\n{err}")


if __name__ == "__main__":
    print(build(force=True, verbose=True))
