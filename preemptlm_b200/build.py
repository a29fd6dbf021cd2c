"""Build libsg_b200.so (every CUDA source of the package) for sm_100a, and the
Python binding of the attention block's entry points, in-tree.

    python -m preemptlm_b200.build          # or __graft_entry__.build()

nvcc cross-compiles without a GPU.  Objects go to ``_build/`` at the repo root;
the shared library goes to ``preemptlm_b200/lib/libsg_b200.so``, the binding
(C++ against the installed torch) to ``preemptlm_b200/_native.so``.  The library
does not need the binding: one that does not compile is a warning, and the calls
that go through it raise until it is built.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB_PATH = LIB_DIR / "libsg_b200.so"
BUILD_DIR = ROOT / "_build"
BINDING_SRC = CSRC / "binding.cpp"
BINDING_PATH = PKG / "_native.so"
BINDING_STAMP = BUILD_DIR / "binding.txt"  # what the binding was built for

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMMON_FLAGS = [
    "-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3", "-DSG_BUILT_ARCH=1000",
    f"-I{ROOT / 'include'}", f"-I{CSRC}",
]


def nvcc() -> str:
    cand = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libsg_b200.so")
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _older(target: Path, inputs: list[Path]) -> bool:
    return not target.exists() or target.stat().st_mtime < max(f.stat().st_mtime for f in inputs)


def _headers() -> list[Path]:
    return [*(ROOT / "include").glob("*.h"), Path(__file__)]


def library_is_stale() -> bool:
    return _older(LIB_PATH, [*sources(), *CSRC.glob("*.cuh"), *_headers()])


def _binding_target() -> str:
    """The interpreter and torch that a binding built now is for: it runs with no other."""
    import torch

    return f"{sys.implementation.cache_tag} torch {torch.__version__} {torch.version.git_version}\n"


def binding_is_stale() -> bool:
    return (_older(BINDING_PATH, [BINDING_SRC, *_headers()]) or not BINDING_STAMP.exists()
            or BINDING_STAMP.read_text() != _binding_target())


def is_stale() -> bool:
    return library_is_stale() or binding_is_stale()


def build_binding() -> Path:
    """g++ against the installed torch's headers and libraries.  RuntimeError if it does
    not compile; the binding that was there, built for something else, is gone then."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    incs = [root / "include", root / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
            Path(nvcc()).resolve().parents[1] / "include", ROOT / "include"]
    libs = [root / "lib"]
    BUILD_DIR.mkdir(exist_ok=True)
    tmp = BINDING_PATH.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in incs), str(BINDING_SRC),
           "-o", str(tmp), *(f"-L{i}" for i in libs), "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10",
           "-lc10_cuda"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
        failed = f"g++ failed on {BINDING_SRC.name}:\n{r.stdout}\n{r.stderr}" if r.returncode else None
    except OSError as e:
        failed = f"g++ could not be run: {e}"
    if failed:
        BINDING_PATH.unlink(missing_ok=True)
        raise RuntimeError(failed)
    os.replace(tmp, BINDING_PATH)
    BINDING_STAMP.write_text(_binding_target())
    return BINDING_PATH


def build_library(force: bool = False, verbose: bool = False, extra_flags: list[str] | None = None) -> Path:
    """Bring the library, and the binding beside it, up to date."""
    with ThreadPoolExecutor(max_workers=1) as ex:
        binding = ex.submit(build_binding) if force or binding_is_stale() else None
        if force or library_is_stale():
            _compile_library(verbose, extra_flags)
        try:
            if binding is not None:
                binding.result()
        except RuntimeError as e:
            warnings.warn(f"the binding of the attention block's entry points was not built: {e}", RuntimeWarning, stacklevel=2)
    return LIB_PATH


def _compile_library(verbose: bool, extra_flags: list[str] | None) -> None:
    BUILD_DIR.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)
    cc = nvcc()
    flags = ARCH_FLAGS + COMMON_FLAGS + list(extra_flags or [])

    def compile_one(src: Path) -> Path:
        obj = BUILD_DIR / (src.stem + ".o")
        cmd = [cc, *flags, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, file=sys.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [cc, *ARCH_FLAGS, "-shared", "-Xcompiler", "-fPIC", *map(str, objs), "-o", str(tmp), "-lcuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB_PATH)


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
    sys.exit(not BINDING_PATH.exists())
