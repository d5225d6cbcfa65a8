"""Compile the HIP sources of jasper_amd into jasper_amd/lib/libjasper_amd.so,
and the Python module that takes torch tensors to its cache operators
(csrc/torch_kv.cpp, host code) into jasper_amd/lib/_kv.so.

hipcc cross-compiles for gfx950 without a GPU. Objects go to
jasper_amd/lib/_build/ and are rebuilt when their source or any header in
csrc/ is newer; `force=True` rebuilds everything.

Flags:
  --offload-arch=gfx950            CDNA4 only
  -ffp-contract=off                the only fused multiply-adds are explicit
                                   (__builtin_fmaf) so results are reproducible
  -target-feature -packed-fp32-ops no packed fp32 VALU instructions
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
OBJDIR = LIBDIR / "_build"
LIB = LIBDIR / "libjasper_amd.so"
BINDING = LIBDIR / "_kv.so"
INCLUDE = PKG.parent / "include"

HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")
CXX = os.environ.get("CXX", shutil.which("g++") or "c++")
ROCM = Path(HIPCC).resolve().parent.parent
ARCH = os.environ.get("JASPER_OFFLOAD_ARCH", "gfx950")

COMMON_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-result",
    f"-I{INCLUDE}",
]


def _sources():
    return sorted(CSRC.glob("*.hip"))


def _newest_header_mtime() -> float:
    hs = list(CSRC.glob("*.hpp")) + list(INCLUDE.glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def _compile(src: Path, force: bool, hdr_mtime: float) -> Path:
    obj = OBJDIR / (src.stem + ".o")
    if not force and obj.exists() and obj.stat().st_mtime >= max(src.stat().st_mtime, hdr_mtime):
        return obj
    cmd = [HIPCC, *COMMON_FLAGS, "-c", str(src), "-o", str(obj)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{r.stdout}\n{r.stderr}")
    return obj


def _run(cmd, what: str) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed:\n{r.stdout}\n{r.stderr}")


def _compile_binding(force: bool) -> Path:
    import torch
    from torch.utils.cpp_extension import include_paths
    src, obj = CSRC / "torch_kv.cpp", OBJDIR / "torch_kv.o"
    newest = max(src.stat().st_mtime, (INCLUDE / "jasper_amd.h").stat().st_mtime)
    if force or not obj.exists() or obj.stat().st_mtime < newest:
        _run([CXX, "-O2", "-std=c++17", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
              f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{INCLUDE}",
              *(f"-isystem{p}" for p in (*include_paths(), sysconfig.get_paths()["include"], ROCM / "include")),
              "-c", str(src), "-o", str(obj)], f"{CXX} for {src.name}")
    return obj


def _link_binding(obj: Path) -> None:
    import torch
    tmp = BINDING.with_suffix(".so.tmp")
    _run([CXX, "-shared", "-fPIC", "-o", str(tmp), str(obj), f"-L{LIBDIR}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN",
          f"-L{Path(torch.__file__).parent / 'lib'}", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"],
         f"link of {BINDING.name}")
    os.replace(tmp, BINDING)


def build(force: bool = False, jobs: int | None = None, verbose: bool = True) -> Path:
    OBJDIR.mkdir(parents=True, exist_ok=True)
    hdr = _newest_header_mtime()
    srcs = _sources()
    jobs = jobs or min(8, os.cpu_count() or 4)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        binding = ex.submit(_compile_binding, force)
        objs = list(ex.map(lambda s: _compile(s, force, hdr), srcs))
        binding = binding.result()
    newest = max(o.stat().st_mtime for o in objs)
    if force or not LIB.exists() or LIB.stat().st_mtime < newest:
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    if force or not BINDING.exists() or BINDING.stat().st_mtime < binding.stat().st_mtime:
        _link_binding(binding)
    if verbose:
        print(f"[jasper_amd] built {LIB}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
