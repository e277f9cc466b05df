"""Builds `libmtpk.so` (gfx950) in this directory with hipcc, one object per translation unit, and
`_mtpk_torch.so`, the C++ calls on torch tensors in front of some of its entry points, with g++. The library
needs hipcc alone: where g++, torch or their headers are missing, it is built and the calls are left out
with a warning.

`python build_lib.py` or `build_lib.build()`; `__graft_entry__.build()` calls it. Rebuilds every
time it is called (the build is the compile check), in parallel across translation units.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
LIB = HERE / "libmtpk.so"
TORCH_LIB = HERE / "_mtpk_torch.so"
OBJ_DIR = HERE / "_build"
ARCH = os.environ.get("MTPK_ARCH", "gfx950")
SOURCES = ["mtpk_runtime.hip", "mtpk_moe.hip", "mtpk_router.hip", "mtpk_accept.hip", "mtpk_deltanet.hip",
           "mtpk_rejection.hip", "mtpk_attention.hip", "mtpk_norm.hip", "mtpk_gemm.hip",
           "mtpk_moe_dense.hip", "mtpk_probe.hip", "mtpk_round.hip", "mtpk_attention_masked.hip",
           "mtpk_rotary.hip", "mtpk_blocks.hip"]

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # no packed-fp32 VALU forms in the code object: some have given wrong results on this part
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    path = Path(rocm) / "bin" / "hipcc"
    return str(path) if path.exists() else "hipcc"


def _compile(src: str) -> Path:
    obj = OBJ_DIR / (Path(src).stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, "-c", str(CSRC / src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src}:\n{res.stdout}\n{res.stderr}")
    return obj


def _torch_calls_need() -> str | None:
    """What `build_torch_calls` lacks here, or None."""
    if shutil.which("g++") is None:
        return "g++"
    if importlib.util.find_spec("torch") is None:
        return "torch"
    import torch

    for header in (Path(torch.__file__).resolve().parent / "include" / "torch" / "csrc" / "utils" / "pybind.h",
                   Path(sysconfig.get_paths()["include"]) / "Python.h"):
        if not header.exists():
            return str(header)
    return None


def build_torch_calls() -> None:
    """`_mtpk_torch.so`: host C++ against the installed torch, no device code and no link to libmtpk (its
    entry points' addresses are handed over when it is loaded)."""
    import torch

    root = Path(torch.__file__).resolve().parent
    tmp = TORCH_LIB.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{INCLUDE}", f"-isystem{root / 'include'}",
           f"-isystem{root / 'include' / 'torch' / 'csrc' / 'api' / 'include'}",
           f"-isystem{sysconfig.get_paths()['include']}", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-DTORCH_EXTENSION_NAME=_mtpk_torch", str(CSRC / "mtpk_torch.cpp"), "-o", str(tmp), f"-L{root / 'lib'}",
           "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10"]  # fmt: skip
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for mtpk_torch.cpp:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, TORCH_LIB)


def build(verbose: bool = False) -> Path:
    OBJ_DIR.mkdir(exist_ok=True)
    with ThreadPoolExecutor(max_workers=min(7, len(SOURCES))) as pool:
        lacks = _torch_calls_need()
        calls = None if lacks else pool.submit(build_torch_calls)
        objs = list(pool.map(_compile, SOURCES))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    if calls is None:
        warnings.warn(f"{TORCH_LIB.name} is not built: {lacks} is missing", stacklevel=2)
    else:
        calls.result()
    if verbose:
        print(f"built {LIB}" + ("" if calls is None else f" and {TORCH_LIB.name}"))
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
