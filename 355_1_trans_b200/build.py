"""Build the sm_100a shared library in-tree with nvcc.

    python 355_1_trans_b200/build.py        -> 355_1_trans_b200/_build/libbsgemm_b200.so
                                               355_1_trans_b200/_build/_bsgemm_ops.so

The library is two translation units (csrc/bsgemm.cu, the GEMMs; csrc/ops.cu,
the operators around them), compiled side by side for
``-gencode arch=compute_100a,code=sm_100a`` and linked with the CUDA runtime
static, so the .so has no dependency on the CUDA runtime that torch
bundles; the driver (libcuda) is reached through cudaGetDriverEntryPoint.  The second file holds the operators' Python
entry points (csrc/binding.cpp, g++ against torch's headers).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT_DIR = PKG / "_build"
LIB = OUT_DIR / "libbsgemm_b200.so"
BINDING = OUT_DIR / "_bsgemm_ops.so"
INCLUDE = PKG.parent / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))


def binding_command() -> list[str]:
    import sysconfig
    import torch
    root = Path(torch.__file__).resolve().parent
    libs = root / "lib"
    return [shutil.which("g++") or "g++", "-O2", "-std=c++20", "-shared", "-fPIC", "-fvisibility=hidden",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-I", str(INCLUDE), "-isystem", str(root / "include"),
            "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
            "-isystem", sysconfig.get_paths()["include"], "-isystem", str(Path(nvcc()).resolve().parents[1] / "include"),
            str(CSRC / "binding.cpp"), "-o", str(BINDING.with_suffix(".so.tmp")), "-L", str(OUT_DIR), "-L", str(libs),
            "-lbsgemm_b200", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]


def needs_build() -> bool:
    if not LIB.exists():
        return True
    t = LIB.stat().st_mtime
    return any(s.stat().st_mtime > t for s in sources())


def build_binding(force: bool = False) -> Path:
    inputs = [CSRC / "binding.cpp", *INCLUDE.glob("*.h")]
    if not force and BINDING.exists() and all(s.stat().st_mtime <= BINDING.stat().st_mtime for s in inputs):
        return BINDING
    res = subprocess.run(binding_command(), capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed ({res.returncode})")
    os.replace(BINDING.with_suffix(".so.tmp"), BINDING)
    return BINDING


def build(force: bool = False, verbose: bool = False, extra: list[str] | None = None) -> Path:
    if not force and not needs_build():
        build_binding()
        return LIB
    OUT_DIR.mkdir(parents=True, exist_ok=True)
    env = dict(os.environ)
    # a compiler wrapper in CC/CXX must not leak into nvcc's host compilation
    env.pop("CC", None)
    env.pop("CXX", None)
    flags = [*(extra or []), *(["-Xptxas=-v"] if verbose else []), *ARCH_FLAGS, "-O3", "-std=c++17", "-lineinfo",
             "-Xcompiler", "-fPIC,-fvisibility=hidden", "--expt-relaxed-constexpr",
             "-ccbin", shutil.which("g++") or "g++", "-I", str(INCLUDE)]
    units = sorted(CSRC.glob("*.cu"))
    objects = [OUT_DIR / (u.stem + ".o") for u in units]
    jobs = [subprocess.Popen([nvcc(), *flags, "-c", "-o", str(o), str(u)], stdout=subprocess.PIPE,
                             stderr=subprocess.STDOUT, text=True, env=env) for u, o in zip(units, objects)]
    tmp = LIB.with_suffix(".so.tmp")
    for job in jobs:
        out = job.communicate()[0]
        if verbose or job.returncode != 0:
            sys.stderr.write(out)
    if any(job.returncode for job in jobs):
        raise RuntimeError("nvcc failed")
    res = subprocess.run([nvcc(), *ARCH_FLAGS, "-shared", "-cudart", "static", "-ccbin", shutil.which("g++") or "g++",
                          "-o", str(tmp), *map(str, objects)], capture_output=True, text=True, env=env)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc failed ({res.returncode})")
    os.replace(tmp, LIB)
    build_binding(force)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
