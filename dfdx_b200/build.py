"""Builds libdfdx_b200.so (sm_100a only) in-tree with nvcc.

    python -m dfdx_b200.build            # incremental
    python -m dfdx_b200.build --force

Each .cu is compiled to an object in `dfdx_b200/lib/obj/` (in parallel), then linked into
`dfdx_b200/lib/libdfdx_b200.so` with a statically linked CUDA runtime.  The driver API is not linked:
the one driver entry point the library needs (tensor-map encoding) is resolved at run time, so the
library loads on a machine without a GPU driver.

`py_heads.cpp`, the host side of heads.py, becomes a Python module in `dfdx_b200/lib/` (g++, against torch's headers), named
after the torch and Python whose binary interface it has, so that no other ones load it; it calls the library through addresses
that it is given and is not linked to it.  Where it cannot be built (no C++ headers of
Python or torch) the library is made all the same, with a warning; the calls of heads.py then raise.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
OBJDIR = LIBDIR / "obj"
LIB = LIBDIR / "libdfdx_b200.so"
SOURCES = ["api.cu", "gemm_simt.cu", "gemm_tc.cu", "gemm_tc_pair.cu", "conv2d.cu", "attention.cu", "attention_bwd.cu", "rowwise.cu",
           "rotary.cu", "kv_cache.cu", "kv_attention.cu", "kv_attention_tc.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _deps_mtime() -> float:
    hdrs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + [PKG.parent / "include" / "dfdx_b200.h"]
    return max(p.stat().st_mtime for p in hdrs if p.exists())


def _compile(src: str, force: bool) -> Path:
    obj = OBJDIR / (src.replace(".cu", ".o"))
    srcp = CSRC / src
    if not force and obj.exists() and obj.stat().st_mtime >= max(srcp.stat().st_mtime, _deps_mtime()):
        return obj
    cmd = [_nvcc(), *NVCC_FLAGS, "-c", str(srcp), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    (OBJDIR / (src + ".log")).write_text(res.stdout + res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{res.stdout}\n{res.stderr}")
    return obj


def module_path() -> Path:
    """The compiled host side of heads.py for the running Python and its torch."""
    import torch
    return LIBDIR / f"_heads.torch-{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX')}"


def _build_module(force: bool) -> None:
    import torch
    src, module = CSRC / "py_heads.cpp", module_path()
    if not force and module.exists() and module.stat().st_mtime >= max(src.stat().st_mtime, (PKG.parent / "include" / "dfdx_b200.h").stat().st_mtime):
        return
    module.unlink(missing_ok=True)              # none rather than that of an earlier source
    root = Path(torch.__file__).resolve().parent
    nvcc = Path(_nvcc())
    cuda = nvcc.resolve().parent.parent / "include" if nvcc.is_absolute() else Path("/usr/local/cuda/include")
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda, Path(sysconfig.get_paths()["include"])]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(f"-isystem{p}" for p in include), str(src), "-o", str(module), f"-L{root / 'lib'}", f"-Wl,-rpath,{root / 'lib'}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{res.stdout}\n{res.stderr}")


def build(force: bool = False, verbose: bool = False) -> Path:
    OBJDIR.mkdir(parents=True, exist_ok=True)
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        module = ex.submit(_build_module, force)
        objs = list(ex.map(lambda s: _compile(s, force), SOURCES))
    if force or not LIB.exists() or any(o.stat().st_mtime > LIB.stat().st_mtime for o in objs):
        cmd = [_nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-cudart", "static",
               "-o", str(LIB), *map(str, objs)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    try:
        module.result()
    except (RuntimeError, ImportError, OSError) as e:
        warnings.warn(f"py_heads.cpp, the host side of heads.py, was not built: {e}", RuntimeWarning)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
