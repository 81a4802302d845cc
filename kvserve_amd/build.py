"""Build the gfx950 C-ABI library ``kvserve_amd/libkvserve_amd.so`` with hipcc.

Every ``csrc/*.hip`` file is compiled separately (in parallel) and linked into one
shared library; ``csrc/kvmi_calls.cpp``, host code, becomes the Python module
``kvserve_amd/_calls.so`` that calls it.  Both are built in-tree so they travel with the
source tree.

    python -m kvserve_amd.build
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
INCLUDE = PKG.parent / "include"
LIB = PKG / "libkvserve_amd.so"
CALLS = PKG / "_calls.so"
OBJ = PKG / "_build"

ARCH = "gfx950"
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    # packed-fp32 VALU ops stay disabled: some of their forms have given wrong results now and then
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in VGPRs: the accumulators feed VALU code directly, without
    # v_accvgpr_read copies out of AGPRs
    "-mllvm", "-amdgpu-mfma-vgpr-form=1",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(exe).exists():
        raise RuntimeError("hipcc not found: the ROCm toolchain is required to build kvserve_amd")
    return exe


def _compile(src: Path, defines=()) -> Path:
    obj = OBJ / (src.stem + ".o")
    cmd = [hipcc(), *HIPCC_FLAGS, *(f"-D{d}" for d in defines), f"-I{INCLUDE}", "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed on {src.name}:\n{res.stderr}")
    return obj


def _build_calls() -> None:
    """The Python module over the library: the paged operators' unchecked calls.  Where g++ or
    Python's or torch's headers are missing it is left out, with a warning, and an old one is
    removed: the library is whole without it, and the calls go the slower way through Python."""
    missing = None
    include = Path(sysconfig.get_paths()["include"])
    try:
        import torch
        root = Path(torch.__file__).resolve().parent
    except ImportError:
        missing = "torch"
    else:
        if not (root / "include" / "torch" / "csrc" / "autograd" / "python_variable.h").exists():
            missing = "torch's headers"
    if not (include / "Python.h").exists():
        missing = "Python's headers"
    if shutil.which("g++") is None:
        missing = "g++"
    if missing:
        CALLS.unlink(missing_ok=True)
        warnings.warn(f"{CALLS.name} is not built, {missing} not found: the paged operators' unchecked calls "
                      "take longer on the host", stacklevel=2)
        return
    rocm = Path(hipcc()).resolve().parents[1]
    tmp = CALLS.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root}/include",
           f"-I{root}/include/torch/csrc/api/include", f"-I{rocm}/include", f"-I{include}",
           f"-I{INCLUDE}", str(CSRC / "kvmi_calls.cpp"), "-o", str(tmp), f"-L{PKG}", f"-l:{LIB.name}",
           "-Wl,-rpath,$ORIGIN", f"-L{root}/lib", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python",
           f"-L{rocm}/lib", "-lamdhip64"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on kvmi_calls.cpp:\n{res.stderr}")
    os.replace(tmp, CALLS)


def build(verbose: bool = False, defines=()) -> Path:
    """Compile every HIP source and link the shared library; returns its path.
    `defines`: preprocessor symbols for every source (KVMI_ORDINARY_LAUNCH: the one-pass
    compress launched as an ordinary kernel, for profilers that cannot follow a
    cooperative launch; its waits are bounded either way)."""
    OBJ.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    workers = min(len(sources), int(os.environ.get("MAX_JOBS", "8")))
    with cf.ThreadPoolExecutor(max_workers=workers) as pool:
        objs = list(pool.map(lambda src: _compile(src, defines), sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB)
    _build_calls()
    if verbose:
        print(f"built {LIB}" + (f" and {CALLS.name}" if CALLS.exists() else ""))
    return LIB


if __name__ == "__main__":
    build(verbose=True, defines=["KVMI_ORDINARY_LAUNCH"] if "--ordinary-launch" in sys.argv[1:] else [])
    sys.exit(0)
