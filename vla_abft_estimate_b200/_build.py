"""Build libabft_b200.so in-tree with nvcc for sm_100a, and _paged_host, the
extension that takes Python calls of the paged cache to it.

The library needs nvcc alone. The extension needs g++ and the headers of the
installed torch, and serves that torch and Python only (its file is named after
them); where it cannot be built the library is built all the same, and the
paged cache takes its longer way through ctypes.

Both land in ``vla_abft_estimate_b200/_lib/`` next to the
package so that they travel with the source tree; nothing is installed into
site-packages and nothing is JIT-compiled at import time.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from importlib import metadata
from pathlib import Path
from typing import Optional

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC_DIR = PKG_DIR / "csrc"
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libabft_b200.so"
HOST_SOURCE = CSRC_DIR / "paged_host.cpp"
INCLUDE_DIR = REPO_DIR / "include"

OBJ_DIR = LIB_DIR / "obj"

# Each source with the headers it includes; a source is recompiled when one
# of them is newer than its object.
SOURCES = {
    "abft_api.cu": ["ptx.cuh", "gemm_kernel.cuh", "aux_kernels.cuh"],
    "paged_api.cu": ["ptx.cuh", "paged_index.cuh", "paged_append.cuh", "paged_decode.cuh",
                     "paged_prefill.cuh", "paged_launch.cuh"],
    "paged_draft_api.cu": ["ptx.cuh", "paged_index.cuh", "paged_append.cuh", "paged_decode.cuh",
                           "paged_prefill.cuh", "paged_tree.cuh", "paged_launch.cuh", "paged_draft.cuh"],
}

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists() and shutil.which(cand) is None:
        raise RuntimeError("nvcc not found; set NVCC or put /usr/local/cuda/bin on PATH")
    return cand


def _inputs(source: str) -> list[Path]:
    return [CSRC_DIR / source, *[CSRC_DIR / h for h in SOURCES[source]], INCLUDE_DIR / "abft_b200.h"]


def _newer(out: Path, inputs: list[Path]) -> bool:
    """``out`` exists and is not older than any of ``inputs``."""
    if not out.exists():
        return False
    t = out.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in inputs)


def _torch_version() -> Optional[str]:
    """Of the installed torch, without importing it; None when there is none."""
    try:
        return metadata.version("torch")
    except metadata.PackageNotFoundError:
        return None


def host_path() -> Path:
    """The extension's file for this torch and Python."""
    return LIB_DIR / f"_paged_host.torch-{_torch_version()}.{sysconfig.get_config_var('SOABI')}.so"


def _host_stale() -> bool:
    return _torch_version() is not None and not _newer(host_path(), [HOST_SOURCE, INCLUDE_DIR / "abft_b200.h"])


def is_stale() -> bool:
    return _host_stale() or not all(_newer(LIB_PATH, _inputs(s)) for s in SOURCES)


def _host_cmd(out: Path) -> list[str]:
    """g++ on the extension, against the headers and libraries of the torch
    that is installed (it reads torch tensors without Python's attributes)."""
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    includes = [INCLUDE_DIR, root / "include", root / "include/torch/csrc/api/include", cuda / "include",
                sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[f"-I{i}" for i in includes], str(HOST_SOURCE), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
            "-lc10", "-lc10_cuda", "-o", str(out)]


def _run(cmd: list[str], verbose: bool) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed ({res.returncode}):\n{res.stdout}\n{res.stderr}")
    if verbose and res.stderr:
        print(res.stderr)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if it is missing or older than its sources (the
    sources that changed, side by side, then one link), and the extension of the
    paged cache; a failure of that one is a warning."""
    if not force and not is_stale():
        return LIB_PATH
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    jobs = []
    for src in SOURCES:
        obj = OBJ_DIR / (Path(src).stem + ".o")
        if force or not _newer(obj, _inputs(src)):
            tmp = obj.with_suffix(".o.tmp")
            jobs.append((tmp, obj, [_nvcc(), *NVCC_FLAGS, f"-I{INCLUDE_DIR}", "-c", str(CSRC_DIR / src), "-o", str(tmp)]))
    if verbose:
        for _, _, cmd in jobs:
            cmd.insert(1, "-Xptxas=-v")
            print(" ".join(cmd))
    with ThreadPoolExecutor(len(jobs) + 1) as pool:
        host = pool.submit(_build_host, verbose) if force or _host_stale() else None
        list(pool.map(lambda j: _run(j[2], verbose), jobs))
        for tmp, obj, _ in jobs:
            os.replace(tmp, obj)
        _link(force, verbose)
        try:
            if host is not None:
                host.result()
        except Exception as e:  # no torch, no g++, other headers: the library is complete without it
            warnings.warn(f"the host extension of the paged cache was not built, its calls take the longer way: {e}")
    return LIB_PATH


def _build_host(verbose: bool) -> None:
    tmp = host_path().with_suffix(".so.tmp")
    _run(_host_cmd(tmp), verbose)
    os.replace(tmp, host_path())


def _link(force: bool, verbose: bool) -> None:
    if not force and all(_newer(LIB_PATH, _inputs(s)) for s in SOURCES):
        return
    tmp = LIB_PATH.with_suffix(".so.tmp")
    _run([_nvcc(), *NVCC_FLAGS[:2], "-shared", *[str(OBJ_DIR / (Path(s).stem + ".o")) for s in SOURCES],
          "-o", str(tmp)], verbose)
    os.replace(tmp, LIB_PATH)


if __name__ == "__main__":
    print(build(force=True, verbose=True))
