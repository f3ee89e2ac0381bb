"""Build the in-tree HIP kernel library for gfx950 with an explicit hipcc line.

``python -m smsgate_amd.ops.build`` (also run by ``__graft_entry__.build()``)
compiles every ``csrc/*.hip`` into ``_lib/libsmsgate_kernels.so``.  The
library exposes a plain C ABI and is loaded with ``ctypes`` — no torch C++
headers (fast builds, no ABI coupling, no hipify step) — and every launch
takes the caller's ``hipStream_t`` so it can be captured into a hipGraph.
The build is skipped when the .so is newer than all sources.

One part is built against torch's headers: ``csrc/train_autograd.cpp``, the training
operators' autograd functions, into ``_lib/smsgate_train_autograd.torch-<version>.<interpreter>.so``
(a file for each that it is compiled against).  A small training call is host time, and a
Python Function costs more of it than all its kernels.  It links the kernel library, whose
entries keep their C ABI.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path
from typing import List, Optional

import torch

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
LIBDIR = HERE / "_lib"
LIB = LIBDIR / "libsmsgate_kernels.so"
AUTOGRAD_SRC = CSRC / "train_autograd.cpp"
AUTOGRAD_NAME = "smsgate_train_autograd"
AUTOGRAD = LIBDIR / f"{AUTOGRAD_NAME}.torch-{torch.__version__}{sysconfig.get_config_var('EXT_SUFFIX') or '.so'}"
ARCH = os.environ.get("SMSGATE_OFFLOAD_ARCH", "gfx950")
# what every HIP source is compiled with
FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-munsafe-fp-atomics",
    # MFMA accumulators in VGPRs: the default AGPR form made the GEMM K-loop
    # shuffle its accumulators (68 v_accvgpr_* per 32 MFMAs) and cost the
    # attention kernels one wave of occupancy (scripts/kernel_resources.py)
    "-mllvm",
    "-amdgpu-mfma-vgpr-form=1",
    # no packed-fp32 instructions (v_pk_fma_f32 and its like, which -O3 forms from
    # ordinary float code): some of their forms have given wrong results now and then.
    # The host pass does not know the feature and says so; that warning is harmless
    "-Xclang",
    "-target-feature",
    "-Xclang",
    "-packed-fp32-ops",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm not installed?)")


def sources() -> List[Path]:
    return sorted(CSRC.glob("*.hip"))


def _older(built: Path, deps: List[Path]) -> bool:
    return not built.exists() or any(d.stat().st_mtime > built.stat().st_mtime for d in deps)


def _tmp(built: Path) -> Path:
    """Where ``built`` is written until it is whole: a file of this process, as the ranks of a
    job may build at once."""
    return built.with_name(f"{built.name}.{os.getpid()}.tmp")


def needs_build(lib: Path = LIB) -> bool:
    return _older(lib, sources() + sorted(CSRC.glob("*.hpp")) + [Path(__file__)])


def build(force: bool = False, verbose: bool = False, extra: Optional[List[str]] = None) -> Path:
    if not force and not needs_build():
        return LIB
    LIBDIR.mkdir(parents=True, exist_ok=True)
    tmp = _tmp(LIB)
    cmd = [
        hipcc(),
        *FLAGS,
        "-shared",
        *(extra or []),
        *[str(s) for s in sources()],
        "-o",
        str(tmp),
    ]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


def needs_build_autograd() -> bool:
    return _older(AUTOGRAD, [AUTOGRAD_SRC, *sorted(CSRC.glob("*.hpp")), Path(__file__)])


def build_autograd(force: bool = False, verbose: bool = False) -> Path:
    """``csrc/train_autograd.cpp`` for this interpreter and torch; after :func:`build`, whose
    library it links."""
    if not force and not needs_build_autograd():
        return AUTOGRAD
    root = Path(torch.__file__).resolve().parent
    tmp = _tmp(AUTOGRAD)
    cmd = [
        os.environ.get("CXX", "g++"),
        "-O2",
        "-std=c++17",
        "-fPIC",
        "-shared",
        "-D__HIP_PLATFORM_AMD__=1",  # torch's and HIP's headers on ROCm ask for both
        "-DUSE_ROCM=1",
        f"-DTORCH_EXTENSION_NAME={AUTOGRAD_NAME}",
        f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
        *(x for d in (root / "include", root / "include/torch/csrc/api/include",
                      Path(hipcc()).resolve().parent.parent / "include", sysconfig.get_paths()["include"])
          for x in ("-isystem", str(d))),
        str(AUTOGRAD_SRC),
        "-o",
        str(tmp),
        f"-L{root / 'lib'}",
        "-ltorch",
        "-ltorch_cpu",
        "-ltorch_hip",
        "-lc10",
        "-lc10_hip",
        "-ltorch_python",
        f"-L{LIBDIR}",
        f"-l:{LIB.name}",
        "-Wl,-rpath,$ORIGIN",
    ]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    os.replace(tmp, AUTOGRAD)
    return AUTOGRAD


if __name__ == "__main__":
    p = build(force="--force" in sys.argv, verbose=True)
    print(p)
    print(build_autograd(force="--force" in sys.argv, verbose=True))
