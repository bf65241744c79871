"""Builds libjitcast_b200.so in-tree with nvcc for sm_100a.

Every ``csrc/*.cu`` file is compiled to an object under ``_build/`` (in parallel, skipped when
the object is newer than its sources and headers) and linked into ``libjitcast_b200.so`` next to
this file, so the library travels with the source tree. The CUDA runtime is linked statically.
"""

from __future__ import annotations

import concurrent.futures
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
BUILD = HERE / "_build"
LIB = HERE / "libjitcast_b200.so"
INCLUDE = HERE.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", "-Xptxas",
         "-warn-spills", "-Xptxas", "-v"]

# Registers a thread that kernels have to be launched with: their warpgroups share them out anew (setmaxnreg), and shares that
# do not add up to the launch's would wait for ever. A compiler that gives another number fails here, not in the calls.
REGISTERS = {
    "kv_attention_tc.cu": [(r"kv_attention_tc_kernel\w*Li16ELi(?:64|128)ELi1E", 168),
                           (r"kv_attention_tc_kernel\w*Li4ELi(?:64|128)ELi1E", 128)],
}


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libjitcast_b200.so")
    return path


def _headers() -> list[Path]:
    return sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def _stale(obj: Path, src: Path, deps: list[Path]) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return any(p.stat().st_mtime > t for p in [src, *deps])


def check_registers(name: str, log: str) -> None:
    """Holds the register counts of ptxas's report on source file `name` to REGISTERS."""
    wanted = REGISTERS.get(name, [])
    used = re.findall(r"Compiling entry function '(\w+)'.*?Used (\d+) registers", log, re.S)
    for pattern, count in wanted:
        found = [(f, int(n)) for f, n in used if re.search(pattern, f)]
        wrong = [(f, n) for f, n in found if n != count]
        if wrong or not found:
            raise RuntimeError(f"{name}: {pattern} needs {count} registers a thread, the compiler gave {wrong or 'none'}")


def _compile(src: Path, obj: Path, verbose: bool) -> None:
    cmd = [nvcc(), *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    check_registers(src.name, r.stderr)
    spilled = [line for line in r.stderr.splitlines() if "spilled" in line]
    if spilled:
        print("\n".join(spilled), file=sys.stderr)


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compiles stale objects and relinks the library if anything changed; returns its path."""
    BUILD.mkdir(exist_ok=True)
    deps = _headers()
    sources = sorted(CSRC.glob("*.cu"))
    todo = [(s, BUILD / (s.stem + ".o")) for s in sources if _stale(BUILD / (s.stem + ".o"), s, deps)]
    if todo:
        workers = jobs or min(len(todo), os.cpu_count() or 4)
        with concurrent.futures.ThreadPoolExecutor(workers) as ex:
            list(ex.map(lambda so: _compile(so[0], so[1], verbose), todo))
    objs = [BUILD / (s.stem + ".o") for s in sources]
    if todo or not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
