"""Build libcsn_b200.so in-tree with nvcc for sm_100a.

    python -m csn_b200._build          (with clifford-space-network_b200/ on sys.path)

Each ``csrc/*.cu`` is compiled to an object in ``csrc/_build/`` (in parallel) and the
objects are linked into ``csn_b200/libcsn_b200.so`` with the CUDA runtime linked
statically, so the library depends only on the driver.  ``csrc/csn_torch.cpp``, the PyTorch binding
of the gated block's entry points, is then compiled against the installed torch into
``csn_b200/_gated.so``, which finds the library beside itself.

The build is content-addressed: a SHA-256 over every source, header and the build flags is
compiled into the library (``csn_version()`` ends in ``src <hash>``) and recorded beside it,
so a library whose sources changed since it was linked is rebuilt whatever the file times
say, and a caller can check that the library it loaded is the one these sources make.  The binding is
made for one torch, Python and C++ runtime as well: a second hash over these, its compiler and its flags
is recorded beside it, and where that changes the binding alone is compiled again.
"""
from __future__ import annotations

import concurrent.futures as cf
import hashlib
import os
import shutil
import subprocess
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = ROOT / "csrc"
OBJ = CSRC / "_build"
LIB = PKG / "libcsn_b200.so"
BINDING = PKG / "_gated.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O2"]
CXX_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden"]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build csn_b200")


def sources() -> list:
    return sorted(CSRC.glob("*.cu"))


HASH_FILE = LIB.with_name(LIB.name + ".srchash")
BINDING_HASH_FILE = BINDING.with_name(BINDING.name + ".srchash")
# what the last build() call did: "built" or "reused"
last_action = None


def source_hash() -> str:
    """SHA-256 (first 16 hex digits) over the build flags and every source and header."""
    deps = sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cpp"))
    deps.append(ROOT.parent / "include" / "csn_b200.h")
    h = hashlib.sha256(" ".join(ARCH + FLAGS).encode())
    for p in deps:
        if p.exists():
            h.update(p.name.encode())
            h.update(p.read_bytes())
    return h.hexdigest()[:16]


def _recorded(product: Path, hash_file: Path, key: str) -> bool:
    """Whether `product` is there and was built under `key`."""
    return product.exists() and hash_file.exists() and hash_file.read_text().strip() == key


def _cxx() -> str:
    # the compiler that torch's own libstdc++ goes with, and not $CXX: one that links its runtime statically
    # makes a module whose streams crash beside torch's
    return next((c for c in ("/usr/bin/g++", shutil.which("g++")) if c and Path(c).exists()), "g++")


def _cxx_version(cxx: str) -> str:
    try:
        return subprocess.run([cxx, "--version"], capture_output=True, text=True).stdout
    except OSError:  # the build says so, if there is one to do
        return ""


def binding_key(digest: str) -> str:
    """The hash that _gated.so is recorded under: the sources' (`digest`) and what it is built with and against."""
    import torch
    what = [digest, torch.__version__, str(torch._C._GLIBCXX_USE_CXX11_ABI), str(sysconfig.get_config_var("SOABI")),
            _cxx_version(_cxx()), *CXX_FLAGS]
    return hashlib.sha256("\0".join(what).encode()).hexdigest()[:16]


def _build_binding(key: str) -> None:
    from torch.utils import cpp_extension
    include = [f"-I{p}" for p in cpp_extension.include_paths(device_type="cuda") + [sysconfig.get_paths()["include"]]]
    where = cpp_extension.library_paths(device_type="cuda")
    tmp = BINDING.with_suffix(".so.tmp")
    cxx = _cxx()
    cmd = [cxx, *CXX_FLAGS, *include, str(CSRC / "csn_torch.cpp"), "-o", str(tmp), f"-L{PKG}", "-l:libcsn_b200.so",
           "-Wl,-rpath,$ORIGIN", *[f"-L{p}" for p in where], "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{cxx} failed on csn_torch.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, BINDING)
    BINDING_HASH_FILE.write_text(key + "\n")


def _build_library(digest: str, verbose: bool) -> None:
    nvcc = _nvcc()
    OBJ.mkdir(parents=True, exist_ok=True)

    def compile_one(src: Path) -> Path:
        obj = OBJ / (src.stem + ".o")
        cmd = [nvcc, *ARCH, *FLAGS, f"-DCSN_SOURCE_HASH=\"{digest}\"", "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout, r.stderr)
        return obj

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH, "-shared", "-cudart", "static", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    HASH_FILE.write_text(digest + "\n")


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile every CUDA source and link the shared library, then the binding (each skipped when it was
    built from exactly these sources, the binding also for this torch, Python and compiler)."""
    global last_action
    digest = source_hash()
    key = binding_key(digest)
    last_action = "reused"
    if force or not _recorded(LIB, HASH_FILE, digest):
        _build_library(digest, verbose)
        last_action = "built"
    if last_action == "built" or not _recorded(BINDING, BINDING_HASH_FILE, key):
        _build_binding(key)
        last_action = "built"
    return LIB


if __name__ == "__main__":
    print(build(force=True, verbose=True))
