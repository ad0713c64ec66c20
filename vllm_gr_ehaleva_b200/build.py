"""Build the C-ABI shared library (sm_100a) in-tree.

    python -m vllm_gr_ehaleva_b200.build            # -> vllm_gr_ehaleva_b200/_gr_beam.so

The library is plain CUDA C++ with an extern "C" interface (include/gr_beam.h);
it links the CUDA runtime statically and has no PyTorch dependency.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_NAME = "_gr_beam.so"
LIB_PATH = os.path.join(PKG_DIR, LIB_NAME)
OBJ_DIR = os.path.join(PKG_DIR, "build")
# each source with the headers it includes (besides include/gr_beam.h)
SOURCES = {
    "gr_beam_step.cu": ["gr_device.cuh", "gr_step_ws.cuh", "gr_step_select_ws.cuh", "gr_nvtx.h"],
    "gr_suffix_kv.cu": ["gr_nvtx.h"],
    "gr_remux.cu": ["gr_nvtx.h"],
    "gr_paged_kv.cu": ["gr_nvtx.h"],
    "gr_paged_attn.cu": ["gr_device.cuh", "gr_nvtx.h"],
}
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    cand = shutil.which("nvcc")
    if cand:
        return cand
    home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    p = os.path.join(home, "bin", "nvcc")
    if os.path.exists(p):
        return p
    raise RuntimeError("nvcc not found (set CUDA_HOME)")


def _inputs(source=None):
    files = []
    for src, headers in SOURCES.items():
        if source is None or src == source:
            files += [os.path.join(CSRC, f) for f in [src, *headers]]
    files.append(os.path.join(ROOT, "include", "gr_beam.h"))
    return files


def _newer(target, files) -> bool:
    if not os.path.exists(target):
        return False
    t = os.path.getmtime(target)
    return all(os.path.getmtime(f) <= t for f in files if os.path.exists(f))


def up_to_date() -> bool:
    return _newer(LIB_PATH, _inputs())


def _run(cmd):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed ({res.returncode}):\n{res.stderr}")
    return res.stderr


def build(force: bool = False, verbose: bool = False, extra_flags=None) -> str:
    """Compiles the sources side by side (those whose object is older than what
    it is made of; all of them with `force` or extra flags) and links them.
    Objects made with extra flags live in a directory of their own for the time
    of the call: none is left for another build to take for its own."""
    if not force and not extra_flags and up_to_date():
        return LIB_PATH
    os.makedirs(OBJ_DIR, exist_ok=True)
    flags = [*ARCH_FLAGS, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-I", os.path.join(ROOT, "include")]
    if verbose:
        flags += ["-Xptxas", "-v"]
    flags += list(extra_flags or [])
    obj_dir = tempfile.mkdtemp(prefix="extra_", dir=OBJ_DIR) if extra_flags else OBJ_DIR

    def compile_one(src):
        obj = os.path.join(obj_dir, src + ".o")
        if not force and not extra_flags and _newer(obj, _inputs(src)):
            return obj, ""
        log = _run([nvcc_path(), *flags, "-c", os.path.join(CSRC, src), "-o", obj + ".tmp.o"])
        os.replace(obj + ".tmp.o", obj)
        return obj, log

    try:
        with ThreadPoolExecutor(len(SOURCES)) as pool:
            done = list(pool.map(compile_one, SOURCES))
        if verbose:
            sys.stderr.write("".join(log for _, log in done))
        _run([nvcc_path(), *ARCH_FLAGS, "-shared", "-o", LIB_PATH + ".tmp", *[obj for obj, _ in done]])
        os.replace(LIB_PATH + ".tmp", LIB_PATH)
    finally:
        if extra_flags:
            shutil.rmtree(obj_dir, ignore_errors=True)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
