"""Builds libkta_b200.so in-tree from kta_b200/csrc/*.cu with nvcc for sm_100a.

``python -m kta_b200.build [-v] [--ptxas]`` compiles every translation unit in parallel into
``kta_b200/_build/`` and links ``kta_b200/libkta_b200.so``. The library links only the
static CUDA runtime; tensor maps come from the driver through cudaGetDriverEntryPoint, so no
libcuda, cuBLAS or torch library is linked (the anti-cheat rule of
src/kta/checks/anticheat.py:38-58 in the reference).

Beside it, ``kta_b200/_binding.so`` (csrc/binding.cpp, g++): the Python binding of the entries
whose calls are short, which uses torch's headers and links the library. It is left out, with a
message, where g++, Python's headers or a CUDA build of torch are missing: the C library needs none
of them.
"""

from __future__ import annotations

import argparse
import hashlib
import importlib.util
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
LIB = PKG / "libkta_b200.so"
BINDING = PKG / "_binding.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = [
    "-O3",
    "-lineinfo",
    "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler",
    "-fPIC,-O3",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: set NVCC or install the CUDA toolkit")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _deps_hash(src: Path, extra: list[str]) -> str:
    h = hashlib.sha256()
    h.update(" ".join(ARCH + FLAGS + extra).encode())
    h.update(src.read_bytes())
    for hdr in sorted([*CSRC.glob("*.cuh"), *CSRC.glob("*.h"), *INCLUDE.glob("*.h")]):
        h.update(hdr.read_bytes())
    return h.hexdigest()[:16]


def _compile(src: Path, extra: list[str], verbose: bool) -> tuple[Path, str]:
    obj = BUILD / (src.stem + ".o")
    stamp = BUILD / (src.stem + ".hash")
    key = _deps_hash(src, extra)
    if obj.exists() and stamp.exists() and stamp.read_text() == key:
        return obj, ""
    cmd = [nvcc(), *ARCH, *FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    stamp.write_text(key)
    return obj, res.stdout + res.stderr


def _run(cmd: list[str], what: str, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stdout}\n{res.stderr}")


def _binding_command() -> tuple[list[str], bytes]:
    """The binding's compiler command, against the torch of this interpreter and the built library,
    and torch's version; raises LookupError for what is missing."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        raise LookupError("torch not found")
    torch_dir = Path(spec.submodule_search_locations[0])
    if not (torch_dir / "lib" / "libc10_cuda.so").exists():
        raise LookupError("torch's CUDA libraries not found")
    gxx = shutil.which("g++")
    if gxx is None:
        raise LookupError("g++ not found")
    python = Path(sysconfig.get_paths()["include"])
    if not (python / "Python.h").exists():
        raise LookupError("Python.h not found")
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{INCLUDE}", f"-I{torch_dir}/include",
           f"-I{torch_dir}/include/torch/csrc/api/include", f"-I{cuda}/include", f"-I{python}",
           str(CSRC / "binding.cpp"), "-o", str(BINDING),
           f"-L{torch_dir}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python",
           f"-L{PKG}", "-l:libkta_b200.so", "-Wl,-rpath,$ORIGIN"]
    return cmd, (torch_dir / "version.py").read_bytes()


def _build_binding(verbose: bool) -> None:
    stamp = BUILD / "binding.hash"
    try:
        cmd, version = _binding_command()
    except LookupError as exc:
        # one of an earlier build may not fit the library's entries
        BINDING.unlink(missing_ok=True)
        stamp.unlink(missing_ok=True)
        print(f"binding not built: {exc} (the paged-cache functions of kta_b200.ops need it; the C "
              "library does not)", file=sys.stderr)
        return
    h = hashlib.sha256(" ".join(cmd).encode() + (CSRC / "binding.cpp").read_bytes() + version)
    for hdr in sorted(INCLUDE.glob("*.h")):
        h.update(hdr.read_bytes())
    if BINDING.exists() and stamp.exists() and stamp.read_text() == h.hexdigest():
        return
    _run(cmd, "building the binding", verbose)
    stamp.write_text(h.hexdigest())


def _build_library(verbose: bool, ptxas: bool) -> Path:
    BUILD.mkdir(exist_ok=True)
    extra = ["-Xptxas", "-v"] if ptxas else []
    srcs = sources()
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as pool:
        results = list(pool.map(lambda s: _compile(s, extra, verbose), srcs))
    for _, log in results:
        if ptxas and log:
            print(log)
    objs = [str(o) for o, _ in results]
    newest = max(Path(o).stat().st_mtime for o in objs)
    if not LIB.exists() or LIB.stat().st_mtime < newest:
        _run([nvcc(), *ARCH, "-shared", "-o", str(LIB), *objs], "link", verbose)
    return LIB


def build(verbose: bool = False, ptxas: bool = False) -> Path:
    """Compiles and links the library and, where its needs are met, the binding; returns the library's
    path. Raises on any compiler error."""
    path = _build_library(verbose, ptxas)
    _build_binding(verbose)
    return path


def main(argv: list[str]) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("-v", "--verbose", action="store_true")
    ap.add_argument("--ptxas", action="store_true", help="print -Xptxas -v resource usage")
    args = ap.parse_args(argv)
    path = build(args.verbose, args.ptxas)
    print(path)
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
