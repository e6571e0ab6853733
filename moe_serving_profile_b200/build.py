"""Build the sm_100a shared library ``libb200moe.so`` and the torch binding
``_ext.so`` next to this file.

nvcc compiles every kernel for ``sm_100a`` only (no PTX fallback, no other
architecture). The library links the CUDA runtime statically and exports the
C ABI declared in ``include/b200moe.h``; the binding calls it (g++, no CUDA
code of its own). Run ``python -m
moe_serving_profile_b200.build`` or call :func:`build`.
"""

from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libb200moe.so"
EXT = PKG / "_ext.so"
SOURCES = ["api.cu", "router.cu", "permute.cu", "gemm.cu", "decode.cu", "combine.cu", "a2a.cu", "a2a_p2p.cu", "p2p.cu", "w8a8.cu",
           "route.cu", "norm.cu", "int8.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    return str(Path(cuda) / "bin" / "nvcc")


def _stale() -> bool:
    if not LIB.exists():
        return True
    built = LIB.stat().st_mtime
    deps = [CSRC / s for s in SOURCES] + list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh"))
    deps.append(INCLUDE / "b200moe.h")
    return any(p.stat().st_mtime > built for p in deps)


def ext_key() -> str:
    """What the torch binding is built for; the binding holds its own as ``built_for``."""
    import sysconfig

    import torch

    return f"torch {torch.__version__} {sysconfig.get_config_var('SOABI')}"


def _ext_stale() -> bool:
    if not EXT.exists():
        return True
    built = EXT.stat().st_mtime
    return (any(p.stat().st_mtime > built for p in (CSRC / "ext.cpp", INCLUDE / "b200moe.h"))
            or ext_key().encode() + b"\0" not in EXT.read_bytes())


def build_ext(force: bool = False) -> Path:
    """Compile the torch binding if its source or the header is newer, or if it
    was built for another torch or Python."""
    if not force and not _ext_stale():
        return EXT
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    tmp = EXT.with_suffix(".so.tmp")
    subprocess.run([
        "g++", "-O2", "-std=c++17", "-fPIC", "-shared", f'-DB200MOE_BUILT_FOR="{ext_key()}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        "-I", str(root / "include"), "-I", str(root / "include" / "torch" / "csrc" / "api" / "include"),
        "-I", sysconfig.get_paths()["include"], "-I", str(Path(nvcc()).parents[1] / "include"), "-I", str(INCLUDE),
        str(CSRC / "ext.cpp"), "-o", str(tmp), "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu",
        "-ltorch_cuda", "-ltorch_python", "-L", str(PKG), f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(tmp, EXT)
    return EXT


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile the library if any source is newer than it, then the binding;
    return the library's path."""
    if not force and not _stale():
        build_ext()
        return LIB
    objs = []
    build_dir = PKG / "_build"
    build_dir.mkdir(exist_ok=True)
    for src in SOURCES:
        obj = build_dir / (Path(src).stem + ".o")
        cmd = [
            nvcc(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
            "-Xptxas", "-v" if verbose else "-O3",
            "-I", str(INCLUDE), "-I", str(CSRC),
            "-c", str(CSRC / src), "-o", str(obj),
        ]
        subprocess.run(cmd, check=True)
        objs.append(str(obj))
    tmp = LIB.with_suffix(".so.tmp")
    subprocess.run([nvcc(), *ARCH, "-shared", "-o", str(tmp), *objs, "-lcudart_static", "-lrt",
                    "-lpthread", "-ldl"], check=True)
    os.replace(tmp, LIB)
    build_ext(force)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(LIB)
