"""Build libsvla.so in-tree with nvcc for sm_100a, and _torch_serving.so, the torch side of the serving operators, with
the host compiler.

    python -m smolvla_mujoco_libero_b200.build [--debug]

Both land next to this file so that they travel with the source tree.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OUT = PKG / "libsvla.so"
TORCH_SRC = CSRC / "torch_serving.cpp"
TORCH_OUT = PKG / "_torch_serving.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


BUILD = PKG / "_build"
HEADER = PKG.parent / "include" / "svla.h"
FLAGS = [*ARCH, "-lineinfo", "-O3", "-std=c++17", "-Xcompiler", "-fPIC"]


def units() -> list[tuple[Path, list[Path]]]:
    """(source, the files its object depends on) for every translation unit of the library."""
    shared = [CSRC / "host.cuh", CSRC / "ptx.cuh", HEADER]
    serving = [CSRC / f"{n}.cuh" for n in ("kv_append", "paged_attention", "packed_attention", "packed_attention_tc",
                                           "serving_common")]
    answer = [CSRC / f"{n}.cuh" for n in ("answer_host", "linear_i8", "quant_rows", "sample")]
    path = [p for p in sorted(CSRC.glob("*.cuh")) if p not in serving + answer]
    return [(CSRC / "svla.cu", [CSRC / "svla.cu", *path, HEADER]),
            (CSRC / "serving.cu", [CSRC / "serving.cu", *serving, *shared]),
            *[(CSRC / n, [CSRC / n, *answer, CSRC / "serving_common.cuh", *shared]) for n in ("answer.cu", "sample.cu")],
            (CSRC / "engine.cpp", [CSRC / "engine.cpp", HEADER])]


def sources() -> list[Path]:
    return sorted({p for _, deps in units() for p in deps} | {TORCH_SRC})


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(p.stat().st_mtime > t for p in deps)


def torch_tag() -> str:
    """What _torch_serving.so is bound to; the module holds it as a string."""
    import torch
    return f"built for torch {torch.__version__}, {sys.implementation.cache_tag}"


def torch_module_fits() -> bool:
    """Whether _torch_serving.so is one of this torch and Python; it is read, not loaded."""
    return TORCH_OUT.exists() and torch_tag().encode() + b"\0" in TORCH_OUT.read_bytes()


def _torch_current() -> bool:
    return not _stale(TORCH_OUT, [TORCH_SRC, HEADER]) and torch_module_fits()


def up_to_date() -> bool:
    return not _stale(OUT, [p for p in sources() if p != TORCH_SRC]) and _torch_current()


def build_torch(force: bool = False) -> Path:
    """_torch_serving.so: a Python module against this torch's headers (no device code)."""
    if not force and _torch_current():
        return TORCH_OUT
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include",
               sysconfig.get_paths()["include"]]
    # g++, as nvcc takes it, with the process's own libstdc++ (a compiler named by $CXX may link another one statically,
    # whose stream facets do not mix with it)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
                    f"-DTORCH_EXTENSION_NAME={TORCH_OUT.stem}", "-DTORCH_API_INCLUDE_EXTENSION_H",
                    f'-DSVLA_TORCH_TAG="{torch_tag()}"',
                    f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                    *[a for p in include for a in ("-isystem", str(p))], "-o", str(TORCH_OUT), str(TORCH_SRC),
                    f"-L{root / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch", "-ltorch_python"], check=True)
    return TORCH_OUT


def build(force: bool = False, debug: bool = False, verbose: bool = False) -> Path:
    if not force and not debug and up_to_date():
        return OUT
    BUILD.mkdir(exist_ok=True)
    objs = []
    for src, deps in units():
        obj = BUILD / (src.stem + (".debug.o" if debug else ".o"))
        if force or debug or _stale(obj, deps):
            cmd = [nvcc(), *FLAGS, "-c", "-o", str(obj), str(src)]
            if debug:
                cmd.insert(1, "-DSVLA_BOUNDS_CHECK")
            if verbose:
                cmd.append("-Xptxas=-v")
            subprocess.run(cmd, check=True)
        objs.append(str(obj))
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", str(OUT), *objs], check=True)
    build_torch(force)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--debug", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, debug=a.debug, verbose=a.verbose))
    sys.exit(0)
