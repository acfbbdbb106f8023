"""Builds liblsrm_hip.so (the gfx950 kernels and their C ABI) and the eager
PyTorch binding _native.so in-tree.

Each ``csrc/*.hip`` file is compiled with hipcc for gfx950 into ``_build/``
and the objects are linked into ``lsrm_hip/liblsrm_hip.so`` next to this
file; ``csrc/torch_binding.cpp`` (host code) is compiled with g++ against the
installed torch and linked to it as ``lsrm_hip/_native.so``.  Usage: ``python -m lsrm_hip.build`` from the package directory, or
``build()`` from Python.
"""

from __future__ import annotations

import concurrent.futures
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent            # .../lsrm_hip
ROOT = PKG_DIR.parent                                # package root
CSRC = ROOT / "csrc"
INCLUDE = ROOT.parent / "include"
BUILD_DIR = ROOT / "_build"
LIB_NAME = "liblsrm_hip.so"
LIB_PATH = PKG_DIR / LIB_NAME
NATIVE_PATH = PKG_DIR / "_native.so"
ARCH = "gfx950"

# Packed fp32 VALU forms are disabled: the compiler would otherwise form
# v_pk_{add,mul,fma}_f32 from plain float code.  MFMA results are kept in
# ordinary VGPRs (gfx950 reads and writes MFMA operands from the unified
# register file); the AGPR form made the compiler copy every score and output
# accumulator between register files on each key tile.
HIP_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-amdgpu-mfma-vgpr-form",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: the HIP toolchain is required to build liblsrm_hip.so")


def _compile(src: Path, obj: Path, extra: list[str]) -> None:
    cmd = [hipcc(), *HIP_FLAGS, *extra, "-c", str(src), "-o", str(obj)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{res.stdout}\n{res.stderr}")


def _run(cmd: list[str], what: str) -> None:
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{res.stdout}\n{res.stderr}")


def _rocm() -> Path:
    return Path(hipcc()).resolve().parents[1]


def _compile_binding(src: Path, obj: Path) -> None:
    import torch

    inc = Path(torch.__file__).resolve().parent / "include"
    _run(["g++", "-std=c++17", "-O2", "-fPIC", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
          "-isystem", str(inc), "-isystem", str(inc / "torch/csrc/api/include"),
          "-isystem", str(_rocm() / "include"),
          "-isystem", sysconfig.get_paths()["include"], "-c", str(src), "-o", str(obj)],
         f"g++ for {src.name}")


def _link_binding(obj: Path) -> None:
    import torch

    lib = Path(torch.__file__).resolve().parent / "lib"
    tmp = NATIVE_PATH.with_suffix(".so.tmp")
    _run(["g++", "-shared", str(obj), "-o", str(tmp), f"-L{PKG_DIR}", "-llsrm_hip", f"-L{lib}",
          "-Wl,--as-needed", "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_hip",
          "-ltorch_hip", f"-L{_rocm() / 'lib'}", "-lamdhip64", "-Wl,-rpath,$ORIGIN"],
         "link of the torch binding")
    os.replace(tmp, NATIVE_PATH)


def build(verbose: bool = False, jobs: int | None = None, extra: list[str] | None = None) -> Path:
    """Compiles every csrc/*.hip for gfx950 and links liblsrm_hip.so, and the
    torch binding against it."""
    extra = list(extra or [])
    BUILD_DIR.mkdir(exist_ok=True)
    sources = sorted(CSRC.glob("*.hip"))
    if not sources:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    objs = [BUILD_DIR / (s.stem + ".o") for s in sources]
    jobs = jobs or min(len(sources), max(1, (os.cpu_count() or 4)))
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as ex:
        futs = [ex.submit(_compile, s, o, extra) for s, o in zip(sources, objs)]
        binding = BUILD_DIR / "torch_binding.obj"
        futs.append(ex.submit(_compile_binding, CSRC / "torch_binding.cpp", binding))
        for f in futs:
            f.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    _link_binding(binding)
    if verbose:
        print(f"built {LIB_PATH} and {NATIVE_PATH}")
    return LIB_PATH


if __name__ == "__main__":
    build(verbose=True, extra=sys.argv[1:])
