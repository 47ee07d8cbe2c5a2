"""Build step for the nova_b200 CUDA library: compiles every ``csrc/*.cu`` for
sm_100a with nvcc and links ``nova_b200/libnova_b200.so`` in the source tree
(the shared object travels with the checkout; nothing goes to site-packages).

The Python binding of the serving operators (``csrc/binding.cpp`` ->
``nova_b200/_fast.so``) is compiled with the host compiler against this torch.

    python -m nova_b200.build            # incremental
    python -m nova_b200.build --force    # rebuild everything
    python -m nova_b200.build --verbose  # show -Xptxas -v register / spill report
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
OBJ = PKG / "_build"
LIB = PKG / "libnova_b200.so"
FAST = PKG / "_fast.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
              "-Xcompiler", "-fvisibility=hidden"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _deps_mtime() -> float:
    files = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    return max((f.stat().st_mtime for f in files), default=0.0)


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.cu"))
    hdr_t = _deps_mtime()
    objs = []
    for src in sources:
        obj = OBJ / (src.stem + ".o")
        objs.append(obj)
        if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, hdr_t):
            continue
        cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{res.stdout}\n{res.stderr}")
        if verbose and res.stderr:
            print(res.stderr, file=sys.stderr)
    if force or not LIB.exists() or LIB.stat().st_mtime < max(o.stat().st_mtime for o in objs):
        cmd = [nvcc(), *ARCH, "-shared", "-o", str(LIB), *map(str, objs), "-cudart", "static"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    build_binding(force)
    return LIB


def build_binding(force: bool = False) -> Path:
    """``nova_b200/_fast.so``, linked to the CUDA library beside it."""
    src = CSRC / "binding.cpp"
    deps = max(src.stat().st_mtime, (INCLUDE / "nova_b200.h").stat().st_mtime, Path(__file__).stat().st_mtime)
    import torch

    # torch's C++ interface and Python's differ between versions: built for others it may load and then misbehave
    built_for = f"torch {torch.__version__}, python {sys.version}"
    OBJ.mkdir(exist_ok=True)
    stamp = OBJ / "fast.built_for"
    if (not force and FAST.exists() and FAST.stat().st_mtime >= deps and stamp.exists()
            and stamp.read_text() == built_for):
        return FAST
    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    includes = [root / "include", root / "include/torch/csrc/api/include", sysconfig.get_paths()["include"], cuda / "include"]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{i}" for i in includes), str(src),
           "-o", str(FAST), f"-L{PKG}", "-l:libnova_b200.so", f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu",
           "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{cmd[0]} failed on {src.name}:\n{res.stdout}\n{res.stderr}")
    stamp.write_text(built_for)
    return FAST


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
