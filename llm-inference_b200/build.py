"""Build libb200attn.so (the C-ABI CUDA library) in-tree for sm_100a.

    python llm-inference_b200/build.py [--force] [--verbose]

Each CUDA translation unit under csrc/ is compiled by nvcc with
``-gencode arch=compute_100a,code=sm_100a`` into _build/, then linked with the
static CUDA runtime into b200attn/libb200attn.so. ptxas resource usage
(registers, spills, shared memory) is kept in _build/ptxas.log.
csrc/pycalls.cpp (the Python calls of the paged cache) is compiled by g++ into
b200attn/_native<suffix of this interpreter's extension modules>, after the
library and apart from it: a machine without g++ or Python's headers gets the
library and a message, and another interpreter compiles its own module only.

Freshness is decided by content, not file times: the SHA-256 of the sources,
headers, flags and nvcc version is written to libb200attn.so.sha256 after a
link (that of the module's source, flags and interpreter beside the module),
and a build whose hash differs (or has none) compiles again. build() prints
whether it compiled or reused the library.
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

PKG_ROOT = os.path.dirname(os.path.abspath(__file__))
REPO_ROOT = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
BUILD = os.path.join(PKG_ROOT, "_build")
INCLUDE = os.path.join(REPO_ROOT, "include")
LIB = os.path.join(PKG_ROOT, "b200attn", "libb200attn.so")
PYCALLS = os.path.join(CSRC, "pycalls.cpp")
NATIVE = os.path.join(PKG_ROOT, "b200attn", "_native" + sysconfig.get_config_var("EXT_SUFFIX"))
# source hash of the linked library (written after a successful link)
STAMP = LIB + ".sha256"
NATIVE_STAMP = NATIVE + ".sha256"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-std=c++17", "-O3", "-lineinfo", *ARCH, "-Xcompiler", "-fPIC,-O3",
              "-Xptxas", "-v", f"-I{INCLUDE}", f"-I{CSRC}"]
CXX_FLAGS = ["-std=c++17", "-O2", "-fPIC", "-shared", f"-I{INCLUDE}"]


def _nvcc() -> str:
    for cand in (shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the b200attn CUDA library cannot be built")


def sources() -> list[str]:
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers() -> list[str]:
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hs += [os.path.join(INCLUDE, "b200attn.h")]
    return hs


def _compile(src: str, verbose: bool) -> tuple[str, str]:
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    cmd = [_nvcc(), *NVCC_FLAGS, "-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {os.path.basename(src)}:\n{res.stdout}\n{res.stderr}")
    return obj, res.stderr


def _nvcc_version() -> str:
    res = subprocess.run([_nvcc(), "--version"], capture_output=True, text=True)
    return res.stdout.strip().splitlines()[-1] if res.returncode == 0 and res.stdout else "unknown"


def _hash_files(paths: list[str]) -> "hashlib._Hash":
    h = hashlib.sha256()
    for p in sorted(paths + [os.path.abspath(__file__)]):
        h.update(os.path.relpath(p, REPO_ROOT).encode())
        with open(p, "rb") as f:
            h.update(f.read())
    return h


def source_hash() -> str:
    """SHA-256 over the library's every source and header (path and bytes), the
    compile and link flags, this script and the nvcc version: the identity of a
    build."""
    h = _hash_files(sources() + _headers())
    # flags with this checkout's paths made relative, so the same tree hashes
    # the same on every machine it is copied to
    h.update(" ".join(f.replace(REPO_ROOT, ".") for f in NVCC_FLAGS + ARCH).encode())
    h.update(_nvcc_version().encode())
    return h.hexdigest()


def native_hash() -> str:
    """The same for the module of Python calls: its source, flags and the interpreter's ABI."""
    h = _hash_files([PYCALLS, os.path.join(INCLUDE, "b200attn.h")])
    h.update(" ".join(f.replace(REPO_ROOT, ".") for f in CXX_FLAGS).encode())
    h.update(str(sysconfig.get_config_var("SOABI")).encode())
    return h.hexdigest()


def _stamped(path: str) -> str | None:
    try:
        with open(path) as f:
            return f.read().strip() or None
    except OSError:
        return None


def built_hash() -> str | None:
    """The source hash recorded when the library in the tree was linked."""
    return _stamped(STAMP)


def _library_fresh() -> bool:
    return os.path.exists(LIB) and built_hash() == source_hash()


def _native_fresh() -> bool:
    return os.path.exists(NATIVE) and _stamped(NATIVE_STAMP) == native_hash()


def needs_build() -> bool:
    return not (_library_fresh() and _native_fresh())


def _link(cmd: list[str], what: str, out: str, stamp: str, want: str, verbose: bool) -> None:
    """Run cmd + [-o a file that takes out's place], then write the stamp."""
    tmp = out + f".tmp{os.getpid()}"
    cmd = [*cmd, "-o", tmp]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, out)
    stamp_tmp = stamp + f".tmp{os.getpid()}"
    with open(stamp_tmp, "w") as f:
        f.write(want + "\n")
    os.replace(stamp_tmp, stamp)


def _build_library(verbose: bool) -> None:
    want = source_hash()
    os.makedirs(BUILD, exist_ok=True)
    srcs = sources()
    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        results = list(ex.map(lambda s: _compile(s, verbose), srcs))
    with open(os.path.join(BUILD, "ptxas.log"), "w") as f:
        for (obj, log), src in zip(results, srcs):
            f.write(f"== {os.path.basename(src)}\n{log}\n")
    _link([_nvcc(), "-shared", *ARCH, *[o for o, _ in results]], "link", LIB, STAMP, want, verbose)


def _python_include() -> str:
    return sysconfig.get_paths()["include"]


def _build_native(verbose: bool) -> str | None:
    """None, or why this machine cannot compile the module."""
    if shutil.which("g++") is None:
        return "there is no g++"
    if not os.path.exists(os.path.join(_python_include(), "Python.h")):
        return f"there is no Python.h in {_python_include()}"
    _link(["g++", *CXX_FLAGS, f"-I{_python_include()}", PYCALLS], f"g++ on {os.path.basename(PYCALLS)}", NATIVE,
          NATIVE_STAMP, native_hash(), verbose)
    return None


def build(force: bool = False, verbose: bool = False, quiet: bool = False) -> str:
    """Compile and link when the library is missing or its recorded source
    hash differs from the tree's; otherwise reuse it. Prints which (unless
    quiet), so a run on another machine shows whether it rebuilt."""
    reuse = not force and _library_fresh()
    if not reuse:
        _build_library(verbose)
    if not quiet:
        print(f"b200attn build: {'reused' if reuse else 'compiled'} {os.path.relpath(LIB, REPO_ROOT)} "
              f"(sources {source_hash()[:16]})", flush=True)
    if force or not _native_fresh():
        missing = _build_native(verbose)
        if missing:
            print(f"b200attn build: without {os.path.basename(NATIVE)}, the paged cache's Python calls: {missing}",
                  flush=True)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))
    sys.exit(0)
