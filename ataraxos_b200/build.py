"""Build libstratego_b200.so for sm_100a (``python -m ataraxos_b200.build``).

The library is compiled in-tree with nvcc into ``ataraxos_b200/_lib/`` so it
travels with the source tree; nothing is JIT-compiled at import time.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB_DIR = PKG / "_lib"
LIB_PATH = LIB_DIR / "libstratego_b200.so"
# the debug build: every kernel checks each game record's indices first (SB_DEBUG_BOUNDS)
DEBUG_LIB_PATH = LIB_DIR / "libstratego_b200_debug.so"
SOURCES = [CSRC / f for f in ("sb_kernels.cu", "sb_logprobs.cu", "sb_distill.cu", "sb_policy_small.cu")]
DEPS = SOURCES + [CSRC / "sb_device.cuh", CSRC / "sb_error.h", CSRC / "sb_policy.cuh", INCLUDE / "stratego_b200.h"]

# the policy operators as torch operators: C++ against torch's headers, no CUDA code
TORCH_LIB_PATH = LIB_DIR / "libstratego_b200_torch.so"
TORCH_SOURCE = CSRC / "sb_torch.cpp"
TORCH_STAMP = LIB_DIR / "libstratego_b200_torch.built_with"  # the torch that they were compiled against

COMPILE_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
]
NVCC_FLAGS = [*COMPILE_FLAGS, "-shared"]


def nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise FileNotFoundError("nvcc not found: the CUDA toolkit is needed to build libstratego_b200.so")


def up_to_date(path: Path = LIB_PATH, deps: list[Path] | None = None) -> bool:
    if not path.exists():
        return False
    t = path.stat().st_mtime
    return all(d.stat().st_mtime <= t for d in (DEPS if deps is None else deps))


def _compile(path: Path, extra: list[str], verbose: bool) -> None:
    LIB_DIR.mkdir(exist_ok=True)
    with tempfile.TemporaryDirectory(dir=LIB_DIR) as tmp:
        cmds, objs = [], []
        for src in SOURCES:
            objs.append(str(Path(tmp) / f"{src.stem}.o"))
            cmds.append([nvcc(), *(["-Xptxas=-v"] if verbose else []), *COMPILE_FLAGS, *extra, f"-I{INCLUDE}",
                         "-c", "-o", objs[-1], str(src)])
        lib = Path(tmp) / path.name
        if verbose:
            print("\n".join(" ".join(c) for c in cmds), flush=True)
        with ThreadPoolExecutor(len(cmds)) as pool:  # one nvcc per source file at a time
            for done in pool.map(lambda c: subprocess.run(c), cmds):
                done.check_returncode()
        subprocess.run([nvcc(), *NVCC_FLAGS, "-o", str(lib), *objs], check=True)
        os.replace(lib, path)


def _torch_in_use() -> str:
    import torch

    return f"{torch.__version__} {Path(torch.__file__).resolve().parent} cxx11_abi={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"


def torch_up_to_date() -> bool:
    """The torch operators are newer than their source and were compiled against this torch's headers and ABI."""
    return (up_to_date(TORCH_LIB_PATH, [TORCH_SOURCE, INCLUDE / "stratego_b200.h"])
            and TORCH_STAMP.exists() and TORCH_STAMP.read_text() == _torch_in_use())


def _compile_torch(verbose: bool) -> None:
    import torch

    LIB_DIR.mkdir(exist_ok=True)
    root = Path(torch.__file__).resolve().parent
    tmp = LIB_DIR / f".{TORCH_LIB_PATH.name}.{os.getpid()}.tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(Path(nvcc()).resolve().parent.parent / "include"), str(TORCH_SOURCE), f"-L{root / 'lib'}",
           "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    TORCH_STAMP.unlink(missing_ok=True)  # a build that stops half way is built again
    subprocess.run(cmd, check=True)
    os.replace(tmp, TORCH_LIB_PATH)
    TORCH_STAMP.write_text(_torch_in_use())


def build(force: bool = False, verbose: bool = False, debug: bool = True) -> Path:
    """Build the production library (with ``debug``, the bounds-checking one too) and the torch operators over it."""
    if force or not up_to_date(LIB_PATH):
        _compile(LIB_PATH, [], verbose)
    if debug and (force or not up_to_date(DEBUG_LIB_PATH)):
        _compile(DEBUG_LIB_PATH, ["-DSB_DEBUG_BOUNDS"], verbose)
    if force or not torch_up_to_date():
        _compile_torch(verbose)
    return LIB_PATH


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
