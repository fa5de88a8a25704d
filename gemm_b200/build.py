"""Build steps for the native parts: the CUDA library (nvcc), the torch binding (g++ through
setup.py) and the test-only CPU oracle (gcc).

The reference builds one torch CUDAExtension from a single .cu that includes torch headers
(setup.py:4-24).  Here the kernels and the C-ABI launcher are compiled by nvcc alone into
``gemm_b200/libneogemm.so`` (seconds), and only the thin binding (csrc/binding.cpp) sees torch.
Everything is built in-tree so that the shared objects travel with the source directory.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
ROOT = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libneogemm.so"
OBJ_DIR = ROOT / "build"
ORACLE_DIR = ROOT / "oracle"
ORACLE_LIB = ORACLE_DIR / "liboracle.so"

# Explicit -gencode: plain -arch=sm_100a would also emit generic compute_100 PTX, for which ptxas
# rejects every tcgen05 instruction.
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo", "-DNDEBUG",
    "-Xcompiler", "-fPIC",
]


def _nvcc() -> str:
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        raise RuntimeError("nvcc not found: the CUDA library cannot be built")
    return nvcc


def _newer(target: Path, sources) -> bool:
    if not target.exists():
        return False
    t = target.stat().st_mtime
    return all(Path(s).stat().st_mtime <= t for s in sources)


def library_sources():
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + [ROOT / "include" / "neogemm.h"]


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """nvcc: csrc/*.cu -> gemm_b200/libneogemm.so for sm_100a, one object per source (in
    ``build/``, compiled side by side; only what changed unless ``force``)."""
    if not force and _newer(LIB_PATH, library_sources()):
        return LIB_PATH
    objects, running = [], []
    shared = [p for p in library_sources() if p.suffix != ".cu"]
    OBJ_DIR.mkdir(exist_ok=True)
    for src in sorted(CSRC.glob("*.cu")):
        obj = OBJ_DIR / (src.stem + ".o")
        objects.append(str(obj))
        # The GEMM kernels take minutes to compile and depend on few of the headers.
        headers = [h for h in shared if _includes(src, h)]
        if not force and _newer(obj, [src, *headers]):
            continue
        cmd = [_nvcc(), *NVCC_FLAGS, "-c", "-o", str(obj), str(src)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        running.append((cmd, subprocess.Popen(cmd, cwd=str(ROOT))))
    failed = [cmd for cmd, process in running if process.wait() != 0]
    if failed:
        raise subprocess.CalledProcessError(1, failed[0])
    # With a soname the extension finds the copy that a process has loaded already, even if the file was
    # rebuilt since: two copies would have two sets of overrides and error records.
    subprocess.run([_nvcc(), *NVCC_FLAGS, "-shared", "-Xlinker", "-soname", "-Xlinker", LIB_PATH.name,
                    "-o", str(LIB_PATH), *objects], check=True, cwd=str(ROOT))
    return LIB_PATH


def _includes(src: Path, header: Path, seen=None) -> bool:
    """Whether ``src`` includes ``header``, directly or through another one."""
    seen = set() if seen is None else seen
    for name in re.findall(r'#include "([^"]+)"', src.read_text()):
        path = (src.parent / name).resolve()
        if path == header.resolve():
            return True
        if path not in seen and path.exists():
            seen.add(path)
            if _includes(path, header, seen):
                return True
    return False


def build_oracle(force: bool = False) -> Path:
    """gcc: oracle/gemm_oracle.c -> oracle/liboracle.so (test infrastructure)."""
    src = ORACLE_DIR / "gemm_oracle.c"
    if not force and _newer(ORACLE_LIB, [src]):
        return ORACLE_LIB
    subprocess.run(["gcc", "-O2", "-shared", "-fPIC", "-o", str(ORACLE_LIB), str(src)], check=True)
    return ORACLE_LIB


def extension_path():
    hits = sorted(ROOT.glob("neoGEMM*.so"))
    return hits[0] if hits else None


def build_extension(force: bool = False) -> Path:
    """setup.py build_ext --inplace: csrc/binding.cpp -> neoGEMM.*.so at the repository root."""
    ext = extension_path()
    srcs = [CSRC / "binding.cpp", ROOT / "include" / "neogemm.h", ROOT / "setup.py"]
    if not force and ext is not None and _newer(ext, srcs) and _newer(ext, [LIB_PATH]):
        return ext
    subprocess.run([sys.executable, "setup.py", "-q", "build_ext", "--inplace"], check=True,
                   cwd=str(ROOT))
    ext = extension_path()
    if ext is None:
        raise RuntimeError("setup.py did not produce the neoGEMM extension")
    return ext


def build_all(force: bool = False) -> None:
    build_library(force)
    build_extension(force)
    build_oracle(force)


if __name__ == "__main__":
    build_all(force="--force" in sys.argv)
    print(LIB_PATH, extension_path(), ORACLE_LIB)
