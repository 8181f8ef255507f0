"""Build the in-tree CUDA library `sonic_sampler_b200/_lib/libsonic_b200.so` for sm_100a.

    python -m sonic_sampler_b200.build [--force]

nvcc cross-compiles without a GPU. The library links the CUDA runtime statically, so it
only needs the driver at run time. Beside it lies the CPython module of `csrc/calls.cpp`, which is
built for the installed torch.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
CSRC = PACKAGE_DIR / "csrc"
OUT = PACKAGE_DIR / "_lib" / "libsonic_b200.so"
CALLS = CSRC / "calls.cpp"
# diagnostic variant with per-phase timing stamps (python -m sonic_sampler_b200.phases)
STAMPS_OUT = PACKAGE_DIR / "_lib" / "libsonic_b200_stamps.so"
API = PACKAGE_DIR.parent / "include" / "sonic_b200.h"
EXPORTS = CSRC / "exports.map"
#: translation unit -> the headers it includes (each is compiled on its own, and again only when
#: one of its files is newer than its object)
UNITS = {
    CSRC / "sampler.cu": [CSRC / "common.cuh", CSRC / "host.h", API],
    CSRC / "cache.cu": [CSRC / "host.h", CSRC / "values.cuh", API],
    CSRC / "attention.cu": [CSRC / "attention.h", CSRC / "host.h", API],
    **{CSRC / f"attention_{types}.cu": [CSRC / "attention_kernel.cuh", CSRC / "attention.h", CSRC / "host.h", CSRC / "values.cuh", API]
       for types in ("bf16", "f16", "bf16_e4m3", "f16_e4m3")},
    CSRC / "norm.cu": [CSRC / "host.h", CSRC / "values.cuh", API],
}
SOURCES = list(UNITS)
HEADERS = sorted({h for headers in UNITS.values() for h in headers} | {EXPORTS})

COMPILE_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-cudart", "static",
]
#: flags of single units: the sampler reproduces bf16/fp32 results exactly, so no implicit
#: multiply-add contraction there
UNIT_FLAGS = {CSRC / "sampler.cu": ["--fmad=false"]}
LINK_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-shared", "-Xcompiler", "-fPIC",
    "-cudart", "static",
    "-Xlinker", f"--version-script={EXPORTS}",
]


def nvcc_path() -> str:
    found = shutil.which("nvcc")
    if found:
        return found
    cand = Path(os.environ.get("CUDA_HOME", "/usr/local/cuda")) / "bin" / "nvcc"
    if cand.is_file():
        return str(cand)
    raise RuntimeError("nvcc not found (set CUDA_HOME or put nvcc on PATH)")


def stale(out: Path = OUT, sources: list[Path] = SOURCES + HEADERS) -> bool:
    """Whether `out` is missing, or older than a source or this file (whose flags it was built with)."""
    if not out.is_file():
        return True
    t = out.stat().st_mtime
    return any(p.stat().st_mtime > t for p in (*sources, Path(__file__)))


def calls_path() -> Path:
    """The CPython module for the installed torch (its C++ classes differ between versions) and the running
    interpreter (so does its C interface)."""
    import sysconfig

    import torch

    return PACKAGE_DIR / "_lib" / f"sonic_b200_calls_{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so"


def calls_command() -> list[str]:
    import sysconfig

    import torch

    home = Path(torch.__file__).resolve().parent
    includes = [home / "include", home / "include" / "torch" / "csrc" / "api" / "include",
                Path(nvcc_path()).resolve().parents[1] / "include", sysconfig.get_paths()["include"]]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in includes), str(CALLS),
            f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda"]


def build(force: bool = False, verbose: bool = False, stamps: bool = False) -> Path:
    """Build the product library, or with `stamps` the phase-stamp diagnostic variant."""
    out = STAMPS_OUT if stamps else OUT
    calls = calls_path()
    fresh_calls = not force and not stale(calls, [CALLS, API])
    if fresh_calls and not stale(out):
        return out
    out.parent.mkdir(parents=True, exist_ok=True)
    define = ["-DSONIC_PHASE_STAMPS"] if stamps else []
    objects, commands = [], []
    for source, headers in UNITS.items():
        # objects sit beside the library; only the sampler has a phase-stamp variant
        suffix = "_stamps.o" if stamps and source.name == "sampler.cu" else ".o"
        obj = out.parent / (source.stem + suffix)
        objects.append(obj)
        newest = max(p.stat().st_mtime for p in (source, *headers, Path(__file__)))
        if force or not obj.is_file() or obj.stat().st_mtime < newest:
            commands.append(([nvcc_path(), *COMPILE_FLAGS, *UNIT_FLAGS.get(source, []), *define, "-c", str(source)], obj))
    if not fresh_calls:
        commands.append((calls_command(), calls))

    def run(cmd, target):
        tmp = target.with_suffix(target.suffix + ".tmp")
        cmd = [*cmd, "-o", str(tmp)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        os.replace(tmp, target)

    with ThreadPoolExecutor() as pool:
        list(pool.map(lambda c: run(*c), commands))
    run([nvcc_path(), *LINK_FLAGS, *map(str, objects)], out)
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose=True, stamps="--stamps" in sys.argv))
