"""Build libllada_quant_cuda.so in-tree with nvcc for sm_100a.

    python -m llada_quant_b200.build          # or __graft_entry__.build()

Sources are the ``csrc/*.cu`` files next to this module; the library lands
beside them in the package directory so that it travels with the repository.
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libllada_quant_cuda.so")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
#: sources without device code shared with others: compiled whole, which ``setmaxnreg`` needs
WHOLE = ("fp8_tc.cu",)


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def up_to_date() -> bool:
    if not os.path.exists(LIB):
        return False
    t = os.path.getmtime(LIB)
    deps = sources() + glob.glob(os.path.join(CSRC, "*.cuh")) + [
        os.path.join(os.path.dirname(HERE), "include", "llada_quant.h")]
    return all(os.path.getmtime(d) <= t for d in deps if os.path.exists(d))


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB

    def run(cmd: list[str]) -> None:
        if verbose:
            print(" ".join(cmd))
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("nvcc failed building libllada_quant_cuda.so")

    with tempfile.TemporaryDirectory() as tmp:
        def compile_one(src: str) -> str:
            name = os.path.basename(src)
            obj = os.path.join(tmp, name[:-3] + ".o")
            run([nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", f"-rdc={'false' if name in WHOLE else 'true'}",
                 "-Xcompiler", "-fPIC", "-Xcompiler", "-O3", "--expt-relaxed-constexpr", "-c", src, "-o", obj])
            return obj

        with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
            objs = list(pool.map(compile_one, sources()))
        run([nvcc(), *ARCH, "-rdc=true", "-shared", "-Xcompiler", "-fPIC", "-o", LIB + ".tmp", *objs])
    os.replace(LIB + ".tmp", LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True))
