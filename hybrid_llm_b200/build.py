"""Build the llmyb native library (sm_100a CUDA kernels behind a C ABI).

``python -m hybrid_llm_b200.build`` compiles every ``csrc/*.cu`` file with
nvcc for ``sm_100a`` and links ``hybrid_llm_b200/lib/libllmyb.so``.  Objects
are cached under ``_build/`` and rebuilt only when a source or header is newer.
``csrc/torch/*.cpp`` becomes ``hybrid_llm_b200/lib/llmyb_torch.so``, a Python
module that takes torch tensors and calls the library (g++, torch's headers;
built again when torch or Python change, left out where they are missing).
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB = LIB_DIR / "libllmyb.so"
TORCH_LIB = LIB_DIR / "llmyb_torch.so"
BUILD = PKG.parent / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
    "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the llmyb CUDA library cannot be built")


def _newest_header() -> float:
    heads = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h"))
    return max((h.stat().st_mtime for h in heads), default=0.0)


def _compile(src: Path, obj: Path, verbose: bool) -> None:
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd += ["-Xptxas", "-v"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, file=sys.stderr)


def _torch_missing() -> str:
    """What the tensor-level module cannot be built without and is not there ("": nothing)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return "torch"
    if not (Path(spec.submodule_search_locations[0]) / "include/ATen/ATen.h").exists():
        return "torch's headers"
    if not (Path(sysconfig.get_paths()["include"]) / "Python.h").exists():
        return "Python's headers"
    return "" if shutil.which("g++") else "g++"


def _torch_module(verbose: bool) -> None:
    """The tensor-level module; torch itself is not imported."""
    torch = Path(importlib.util.find_spec("torch").submodule_search_locations[0])
    cuda = Path(nvcc()).resolve().parents[1]
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-I{sysconfig.get_paths()['include']}", f"-isystem{torch / 'include'}",
           f"-isystem{torch / 'include/torch/csrc/api/include'}", f"-isystem{cuda / 'include'}",
           *map(str, sorted((CSRC / "torch").glob("*.cpp"))), "-o", str(tmp),
           f"-L{torch / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           f"-L{LIB_DIR}", "-lllmyb", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on csrc/torch:\n{res.stdout}\n{res.stderr}")
    if verbose and (res.stdout or res.stderr):
        print(res.stdout + res.stderr, file=sys.stderr)
    os.replace(tmp, TORCH_LIB)


def _build_torch_module(force: bool, verbose: bool) -> None:
    """Builds the tensor-level module where it is out of date.  The native library
    and engine do without it: where it cannot be built it is left out (a module
    of older sources would pass another argument block), and loading it raises."""
    stamp = BUILD / "llmyb_torch.stamp"
    missing = _torch_missing()
    want = missing or f"torch {importlib.metadata.version('torch')}, python {sys.version}"
    inputs = [*(CSRC / "torch").glob("*.cpp"), *(PKG.parent / "include").glob("*.h")]
    if (not force and TORCH_LIB.exists() and stamp.exists() and stamp.read_text() == want
            and TORCH_LIB.stat().st_mtime >= max(f.stat().st_mtime for f in inputs)):
        return
    if missing:
        TORCH_LIB.unlink(missing_ok=True)
        print(f"{TORCH_LIB.name} is not built: {missing} not found (the paged cache's Python calls "
              "need it)", file=sys.stderr)
        return
    _torch_module(verbose)
    stamp.write_text(want)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile and link; returns the path of the shared library."""
    BUILD.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    head_t = _newest_header()
    jobs = []
    objs = []
    for src in sources:
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, head_t):
            jobs.append((src, obj))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            for fut in [ex.submit(_compile, s, o, verbose) for s, o in jobs]:
                fut.result()
    if jobs or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart_static", "-lrt",
               "-lpthread", "-ldl"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
        os.replace(tmp, LIB)
    _build_torch_module(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
