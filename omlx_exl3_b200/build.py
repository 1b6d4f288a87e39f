"""Build libexl3b200.so (the C ABI in include/exl3_b200.h) from csrc/*.cu for sm_100a.

    python -m omlx_exl3_b200.build [--force] [--verbose]

Every translation unit is compiled by nvcc with `-gencode arch=compute_100a,code=sm_100a` (the
architecture-specific target: tcgen05 / TMA instructions need the `a` variant), objects go to
omlx_exl3_b200/_build/, and the shared library is linked in-tree next to this file so that it
travels with the repository snapshot. nvcc cross-compiles; no GPU is needed to build.

csrc/exl3_torch.cpp, the native argument checks of the paged-serving calls, is compiled by the host compiler against the
installed torch into _exl3_torch.so beside it; it links libexl3b200.so.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = PKG / "_build"
LIB = PKG / "libexl3b200.so"
BINDING_SRC = CSRC / "exl3_torch.cpp"
BINDING = PKG / "_exl3_torch.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xcompiler", "-fvisibility=hidden", "-DEXL3_BUILD"]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    return cand


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))


def up_to_date() -> bool:
    if not LIB.exists():
        return False
    t = LIB.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in _deps())


def _binding_target() -> str:
    """The torch and interpreter a binding is compiled against, as it carries them in its docstring."""
    import torch
    return f"built for torch {torch.__version__}, {sys.implementation.cache_tag}"


def binding_up_to_date() -> bool:
    return (BINDING.exists() and all(p.stat().st_mtime <= BINDING.stat().st_mtime for p in [BINDING_SRC, Path(__file__), *INCLUDE.glob("*.h")])
            and f"{_binding_target()}\0".encode() in BINDING.read_bytes())


def build_binding(force: bool = False) -> Path:
    """Compile the torch binding (when its source or the installed torch changed); the library has to be there."""
    if not force and binding_up_to_date():
        return BINDING
    import torch
    troot = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent if shutil.which(nvcc()) else Path("/usr/local/cuda")
    tmp = BINDING.with_suffix(f".so.{os.getpid()}.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f'-DEXL3_BUILT_FOR="{_binding_target()}"',
           "-isystem", str(troot / "include"), "-isystem", str(troot / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(cuda / "include"), "-isystem", sysconfig.get_path("include"), f"-I{INCLUDE}",
           str(BINDING_SRC), "-o", str(tmp), f"-L{PKG}", "-lexl3b200", f"-L{troot / 'lib'}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN",
           # the C++ runtime that torch has loaded, whatever the compiler would link: with a second one inside the binding (a
           # toolchain that has only libstdc++.a) a message that formats a number ends the process
           "-nostdlib++", "-l:libstdc++.so.6"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {BINDING_SRC.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)
    return BINDING


def _compile(src: Path, verbose: bool) -> Path:
    obj = BUILD / (src.stem + ".o")
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr:
        print(r.stderr, flush=True)
    return obj


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile (when sources changed) and return the path of libexl3b200.so; the torch binding too."""
    if not force and up_to_date():
        build_binding()
        return LIB
    BUILD.mkdir(exist_ok=True)
    srcs = sources()
    with ThreadPoolExecutor(max_workers=max(1, min(len(srcs), os.cpu_count() or 4))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB.with_suffix(f".so.{os.getpid()}.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    build_binding(force)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
