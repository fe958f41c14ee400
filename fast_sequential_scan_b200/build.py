"""In-tree build of ``libfss_b200.so`` (the C-ABI CUDA library) with plain nvcc for sm_100a, and of
``_fss_torch*.so`` (the autograd side of the entry points, ``csrc/fss_torch*.cpp``) with g++ against torch.
The latter carries the Python and the torch it was compiled for in its name: one for another torch is neither
taken for up to date here nor loaded by the package.

The library needs no libtorch and no pybind: its only inputs are ``csrc/*.cu[h]`` and
``include/fss_b200.h``.  The results sit beside this file so that they travel with the source tree.  Run as
``python fast_sequential_scan_b200/build.py`` (add ``--force`` to rebuild, ``--verbose`` for ptxas
resource usage); run it as a script, not with ``-m``: importing the package needs the library.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJECTS = PKG / "build"      # one object for each .cu, with the list of what it was made from
LIB = PKG / "libfss_b200.so"
TORCH_SOURCES = [CSRC / "fss_torch.cpp", CSRC / "fss_torch_layers.cpp"]

NVCC_FLAGS = [
    "-O3", "-std=c++17",
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found: cannot build libfss_b200.so")
    return exe


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [PKG.parent / "include" / "fss_b200.h"]


def is_stale() -> bool:
    if not LIB.is_file():
        return True
    t = LIB.stat().st_mtime
    return any(s.stat().st_mtime > t for s in sources() + [Path(__file__)])


def torch_lib() -> Path:
    """Where ``fss_torch*.cpp`` are built for the running Python and torch."""
    import torch
    return PKG / f"_fss_torch.{sys.implementation.cache_tag}.torch-{torch.__version__}.so"


def build_torch(force: bool = False) -> Path:
    lib = torch_lib()
    inputs = [*TORCH_SOURCES, CSRC / "fss_torch.h", PKG.parent / "include" / "fss_b200.h", Path(__file__)]
    if not force and lib.is_file() and lib.stat().st_mtime >= max(p.stat().st_mtime for p in inputs):
        return lib
    import sysconfig

    import torch
    root = Path(torch.__file__).resolve().parent
    includes = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", Path(sysconfig.get_paths()["include"]),
                Path(_nvcc()).resolve().parent.parent / "include"]
    cmd = [shutil.which("g++") or "c++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden",
           "-DTORCH_EXTENSION_NAME=_fss_torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *[f"-I{p}" for p in includes], *map(str, TORCH_SOURCES), "-o", str(lib), f"-L{root / 'lib'}",
           f"-Wl,-rpath,{root / 'lib'}", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed building {lib.name}")
    return lib


def _object_is_stale(source: Path, obj: Path) -> bool:
    made_from = obj.with_suffix(".d")
    if not obj.is_file() or not made_from.is_file():
        return True
    t = obj.stat().st_mtime
    names = made_from.read_text().replace("\\\n", " ").split(":", 1)[-1].split()
    return any(not Path(n).is_file() or Path(n).stat().st_mtime > t for n in [str(source), str(Path(__file__)), *names])


def _compile(nvcc: str, source: Path, obj: Path, verbose: bool):
    cmd = [nvcc, *NVCC_FLAGS, *(["-Xptxas", "-v"] if verbose else []), "-MD", "-MF", str(obj.with_suffix(".d")), "-c", str(source), "-o", str(obj)]
    return subprocess.run(cmd, env=dict(os.environ), capture_output=True, text=True)


def build(force: bool = False, verbose: bool = False) -> Path:
    build_torch(force)
    if not force and not is_stale():
        return LIB
    from concurrent.futures import ThreadPoolExecutor
    nvcc = _nvcc()
    OBJECTS.mkdir(exist_ok=True)
    objects = {f: OBJECTS / f"{f.stem}.o" for f in sorted(CSRC.glob("*.cu"))}
    stale = [f for f, o in objects.items() if force or _object_is_stale(f, o)]
    with ThreadPoolExecutor(len(objects)) as pool:
        results = list(pool.map(lambda f: _compile(nvcc, f, objects[f], verbose), stale))
    if not any(r.returncode for r in results):
        results.append(subprocess.run([nvcc, *NVCC_FLAGS, "-shared", "-o", str(LIB), *map(str, objects.values())], capture_output=True, text=True))
    failed = any(r.returncode for r in results)
    if verbose or failed:
        for r in results:
            sys.stderr.write(r.stdout + r.stderr)
    if failed:
        raise RuntimeError("nvcc failed building libfss_b200.so")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
