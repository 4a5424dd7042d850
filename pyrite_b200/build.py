"""Build libpyrite_b200.so in-tree for sm_100a, and the Python calls of its serving kernels.

    python -m pyrite_b200.build          # compile (incremental)
    python -m pyrite_b200.build --force  # rebuild everything

The library is plain CUDA C++ with a C ABI (include/pyrite_b200.h); it links
the CUDA runtime statically, so it needs only the driver at run time.
serving_calls is a CPython module over torch's tensors; its file name carries
the versions it was compiled for.  Without torch or g++ the library is built all
the same, with a warning, and only the serving calls are missing.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import hashlib
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "_native" / "obj"
LIB = PKG / "_native" / "libpyrite_b200.so"
SOURCES = ["capi.cu", "mv_generic.cu", "mv_tile.cu", "mm_tc.cu", "noalloc.cu", "decode.cu", "moe.cu", "allreduce.cu", "paged.cu",
           "paged_attention.cu", "paged_attention_tc.cu", "sampling.cu", "quantize.cpp"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
# host code: no FMA contraction, so the quantizers round exactly like the
# Python encoders they restate
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-ffp-contract=off", "--expt-relaxed-constexpr",
              "-I", str(ROOT / "include")]


def _calls_sources() -> tuple[Path, ...]:
    return CSRC / "serving_calls.cpp", ROOT / "include" / "pyrite_b200.h"


def calls_path() -> Path:
    """The module of the serving calls for this torch, this Python and these sources: one built from others has
    another name and is never loaded."""
    import torch
    key = hashlib.sha256(b"".join(p.read_bytes() for p in _calls_sources())).hexdigest()[:12]
    return PKG / "_native" / f"serving_calls-torch{torch.__version__}-{sys.implementation.cache_tag}-{key}.so"


def nvcc() -> str:
    found = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(found).exists():
        raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libpyrite_b200.so")
    return found


def _headers_mtime() -> float:
    paths = list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))
    return max((p.stat().st_mtime for p in paths), default=0.0)


def _run(cmd: list[str], out: Path, what: str) -> str:
    """Run ``cmd`` for the file ``out``, written under a name of its own and then put in its place: builds at the
    same time (the ranks of one job) each put a whole file there.  Returns what the command wrote to stderr."""
    out.parent.mkdir(parents=True, exist_ok=True)
    fd, tmp = tempfile.mkstemp(prefix=out.name + ".", suffix=out.suffix, dir=out.parent)
    os.close(fd)
    try:
        res = subprocess.run([*cmd, "-o", tmp], capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"{what}:\n{res.stdout}\n{res.stderr}")
        os.chmod(tmp, 0o755 if out.suffix == ".so" else 0o644)
        os.replace(tmp, out)
    finally:
        Path(tmp).unlink(missing_ok=True)
    return res.stderr


def _compile(src: Path, obj: Path, verbose: bool) -> None:
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", str(src)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    said = _run(cmd, obj, f"nvcc failed for {src.name}")
    if verbose and said:
        sys.stderr.write(said)


def build_calls(force: bool = False) -> Path:
    import torch
    src, lib = _calls_sources()[0], calls_path()
    if not force and lib.exists():
        return lib
    home, cuda = Path(torch.__file__).parent, Path(nvcc()).resolve().parent.parent
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", str(src),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", str(home / "include"),
           "-I", str(home / "include/torch/csrc/api/include"), "-I", str(cuda / "include"),
           "-I", sysconfig.get_paths()["include"], "-L", str(home / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
           "-ltorch_python"]
    _run(cmd, lib, f"g++ failed for {src.name}")
    for old in lib.parent.glob(f"serving_calls-torch{torch.__version__}-{sys.implementation.cache_tag}*.so"):
        if old != lib:  # of other sources
            old.unlink(missing_ok=True)
    return lib


def link(objs: list[Path]) -> Path:
    _run([nvcc(), *ARCH, "-shared", *map(str, objs)], LIB, "link failed")
    return LIB


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(parents=True, exist_ok=True)
    hdr = _headers_mtime()
    jobs = []
    for name in SOURCES:
        src, obj = CSRC / name, OBJ / (Path(name).stem + ".o")
        if force or not obj.exists() or obj.stat().st_mtime < max(src.stat().st_mtime, hdr):
            jobs.append((src, obj))
    with cf.ThreadPoolExecutor(max(1, min(len(jobs) + 1, os.cpu_count() or 1))) as pool:
        calls = pool.submit(build_calls, force)
        list(pool.map(lambda j: _compile(*j, verbose), jobs))
        objs = [OBJ / (Path(n).stem + ".o") for n in SOURCES]
        if force or jobs or not LIB.exists():
            link(objs)
        try:
            calls.result()
        except Exception as e:  # noqa: BLE001 - the library needs neither torch nor g++; the serving calls raise when used
            warnings.warn(f"the serving calls (pyrite_b200.kernels.paged, .sampling) were not built: {e}", RuntimeWarning)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true", help="print ptxas resource usage")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
