"""Build recipe for the in-tree HIP library (gfx950 only).

``python -m qwen_image_kernel_amd.build`` (or ``build()``) compiles every
``csrc/*.hip`` file with hipcc into ``lib/libqik_attn.so``.  The library is
written to a temporary name and renamed, so a concurrent reader never sees a
half-written file.
"""

from __future__ import annotations

import concurrent.futures
import glob
import os
import shutil
import subprocess
import sys
import tempfile

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(REPO_DIR, "include")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libqik_attn.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # keep hipcc from forming packed-fp32 VALU ops (v_pk_*_f32)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # every device atomic here is issued by one thread; the atomic optimizer's
    # wave-wide rewrite of such an atomic reads its return value at once,
    # which would make the attention kernel wait out the queue draw's round
    # trip where it means to overlap it with the unit's merge and store
    "-mllvm", "-amdgpu-atomic-optimizer-strategy=None",
    "-Wall",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    cand = os.path.join(ROCM, "bin", "hipcc")
    if os.path.exists(cand):
        return cand
    found = shutil.which("hipcc")
    if not found:
        raise RuntimeError("hipcc not found (set ROCM_PATH)")
    return found


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def build(verbose: bool = False) -> str:
    """Compile the HIP sources into lib/libqik_attn.so and return its path.

    Every source is an object of its own, compiled side by side: the attention
    kernels alone take two minutes."""
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = f"{LIB_PATH}.tmp{os.getpid()}"
    with tempfile.TemporaryDirectory(prefix="qik_build_") as objs:
        def compile_one(src: str) -> str:
            obj = os.path.join(objs, os.path.basename(src) + ".o")
            _run([hipcc(), *HIPCC_FLAGS, "-c", f"-I{INCLUDE}", src, "-o", obj], verbose)
            return obj

        with concurrent.futures.ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
            built = list(pool.map(compile_one, sources()))
        try:
            _run([hipcc(), "--offload-arch=gfx950", "-shared", *built, "-o", tmp,
                  f"-Wl,-rpath,{os.path.join(ROCM, 'lib')}"], verbose)
        except RuntimeError:
            if os.path.exists(tmp):
                os.remove(tmp)
            raise
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed ({res.returncode}):\n{res.stderr}")
    if verbose and res.stderr.strip():
        print(res.stderr, file=sys.stderr)


if __name__ == "__main__":
    print(build(verbose=True))
