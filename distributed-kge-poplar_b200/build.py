"""Compile the engine for sm_100a, in tree.

    python distributed-kge-poplar_b200/build.py [--force] [--verbose]

Produces, next to this file:
  libkge_b200.so              the C ABI of include/kge_b200.h (CUDA runtime only)
  libpoplar_kge<ext-suffix>   the pybind11 module with the reference's `Engine` class
  libkge_torch<ext-suffix>    the operators on device arrays for torch tensors (the only part that knows torch)
A target is rebuilt when any source or header is newer than it, the last one also when torch is another version.
"""

from __future__ import annotations

import argparse
import importlib.metadata
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import Optional

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]

LIB = HERE / "libkge_b200.so"
MODULE = HERE / ("libpoplar_kge" + sysconfig.get_config_var("EXT_SUFFIX"))
TORCH_MODULE = HERE / ("libkge_torch" + sysconfig.get_config_var("EXT_SUFFIX"))


def _newer_than(target: Path, sources) -> bool:
    if not target.exists():
        return True
    stamp = target.stat().st_mtime
    return any(Path(s).stat().st_mtime > stamp for s in sources)


def _run(cmd, verbose: bool) -> None:
    if verbose:
        print(" ".join(str(c) for c in cmd), flush=True)
    proc = subprocess.run([str(c) for c in cmd], capture_output=True, text=True)
    if proc.returncode != 0 or verbose:
        sys.stderr.write(proc.stdout + proc.stderr)
    if proc.returncode != 0:
        raise RuntimeError(f"build step failed: {' '.join(str(c) for c in cmd)}")


def build(force: bool = False, verbose: bool = False) -> None:
    headers = list(CSRC.glob("*.hpp")) + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    lib_sources = sorted(CSRC.glob("*.cu"))
    common = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-Wall,-Wextra", *ARCH]
    if verbose:
        common += ["-Xptxas", "-v"]
    if force or _newer_than(LIB, lib_sources + headers + [Path(__file__)]):
        objects = [HERE / "build" / (src.stem + ".o") for src in lib_sources]
        objects[0].parent.mkdir(exist_ok=True)
        stale = [[NVCC, *common, "-c", src, "-o", obj] for src, obj in zip(lib_sources, objects)
                 if force or _newer_than(obj, [src, *headers, Path(__file__)])]
        with ThreadPoolExecutor() as pool:  # the sources side by side
            list(pool.map(lambda cmd: _run(cmd, verbose), stale))
        _run([NVCC, "-shared", *ARCH, "-o", LIB, *objects, "-cudart", "shared"], verbose)
    binding = CSRC / "pybind_module.cpp"
    if binding.exists() and (force or _newer_than(MODULE, [binding, LIB, *headers])):
        import pybind11

        _run(
            [
                os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall",
                f"-I{pybind11.get_include()}", f"-I{sysconfig.get_paths()['include']}", f"-I{INCLUDE}",
                binding, "-o", MODULE, f"-L{HERE}", "-lkge_b200", "-Wl,-rpath,$ORIGIN",
            ],
            verbose,
        )
    _build_torch_module(force, verbose)


def _torch_version() -> Optional[str]:
    """The installed torch's version, None without one; torch itself is not imported for it."""
    try:
        return importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        return None


def _build_torch_module(force: bool, verbose: bool) -> None:
    """libkge_torch, built anew for another torch than the one it was built for.  Without torch nobody can load it: nothing is built,
    and the parts that need no torch stand by themselves."""
    binding, version = CSRC / "torch_binding.cpp", _torch_version()
    if version is None:
        print("libkge_torch is not built: there is no torch", file=sys.stderr)
        return
    built_for = HERE / "build" / "libkge_torch.version"
    same = built_for.exists() and built_for.read_text() == version
    if not force and same and not _newer_than(TORCH_MODULE, [binding, INCLUDE / "kge_b200.h"]):
        return
    from torch.utils import cpp_extension

    includes = [f"-I{p}" for p in cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"], INCLUDE]]
    torch_libs = [f"-L{p}" for p in cpp_extension.library_paths()]
    _run(
        [
            os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-Wall", "-DTORCH_EXTENSION_NAME=libkge_torch", *includes,
            binding, "-o", TORCH_MODULE, f"-L{HERE}", "-lkge_b200", *torch_libs, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10",
            "-lc10_cuda", "-Wl,-rpath,$ORIGIN",
        ],
        verbose,
    )
    built_for.parent.mkdir(exist_ok=True)
    built_for.write_text(version)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    build(args.force, args.verbose)
    print("built", LIB.name, MODULE.name if MODULE.exists() else "")
