"""Builds libhalo_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU).

    python -m halo_flash_b200.build [--force] [--verbose]

Objects go to halo_flash_b200/csrc/build/, the library to halo_flash_b200/libhalo_b200.so, and beside it the
extension module through which ops.py makes its attention calls (csrc/bind.cpp, host code only).
A source is recompiled when it or any header is newer than its object.
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from importlib.util import find_spec
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
OBJ = CSRC / "build"
LIB = PKG / "libhalo_b200.so"
INCLUDE = PKG.parent / "include"
BIND = PKG / ("_bind" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

SOURCES = ["norm.cu", "norm_odd.cu", "rope.cu", "elementwise.cu", "embed.cu", "quant.cu", "hc.cu", "conv.cu", "paged.cu", "attention.cu", "api.cu", "launch.cu", "static_scratch.cu"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17",
    "-fmad=false",  # multiplies and adds round separately, as the CPU operators do
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: libhalo_b200.so cannot be built (there is no CPU fallback)")


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def _build_bind(nvcc: str, force: bool) -> None:
    """The extension module, where Python's and torch's headers are; a C or C++ program needs neither."""
    spec = find_spec("torch")
    headers = Path(sysconfig.get_paths()["include"])
    if spec is None or not (headers / "Python.h").exists():
        print(f"[build] no {'torch' if spec is None else headers / 'Python.h'}: {BIND.name}, through which ops.py makes its attention calls, is not built",
              file=sys.stderr)
        return
    src = CSRC / "bind.cpp"
    torch = Path(spec.submodule_search_locations[0])
    cuda = Path(nvcc).resolve().parents[1]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", str(INCLUDE), "-I", str(headers),
           "-isystem", str(torch / "include"), "-isystem", str(torch / "include/torch/csrc/api/include"), "-isystem", str(cuda / "include"),
           str(src), "-o", str(BIND), "-L", str(torch / "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
           "-L", str(PKG), "-lhalo_b200", "-Wl,-rpath,$ORIGIN"]
    # a module built against another torch or Python does not load
    made_with, stamp = "\n".join([*cmd, sys.version, (torch / "version.py").read_text()]), OBJ / "bind.stamp"
    if not force and not _stale(BIND, [src, INCLUDE / "halo_b200.h", Path(__file__)]) and stamp.exists() and stamp.read_text() == made_with:
        return
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"g++ failed on bind.cpp:\n{p.stdout}\n{p.stderr}")
    stamp.write_text(made_with)


def build(force: bool = False, verbose: bool = False) -> Path:
    nvcc = _nvcc()
    OBJ.mkdir(parents=True, exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h")) + [Path(__file__)]

    def compile_one(name: str):
        src, obj = CSRC / name, OBJ / (Path(name).stem + ".o")
        if not force and not _stale(obj, [src, *headers]):
            return name, None
        # HALO_B200_NVCC_FLAGS: extra flags for experiments (e.g. -DHALO_PF_HC=0); use --force when it changes
        extra = os.environ.get("HALO_B200_NVCC_FLAGS", "").split()
        cmd = [nvcc, *NVCC_FLAGS, *extra, "-I", str(INCLUDE), "-c", str(src), "-o", str(obj)]
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {name}:\n{p.stdout}\n{p.stderr}")
        (OBJ / (Path(name).stem + ".ptxas.txt")).write_text(p.stderr)
        return name, p.stderr

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, SOURCES))
    rebuilt = [n for n, log in results if log is not None]
    if verbose:
        for n, log in results:
            if log:
                spills = [l for l in log.splitlines() if "spill" in l and "0 bytes spill stores" not in l]
                print(f"[build] {n}: compiled, {len(spills)} kernels with spills")
    objs = [OBJ / (Path(n).stem + ".o") for n in SOURCES]
    if force or rebuilt or _stale(LIB, objs):
        cmd = [nvcc, "-shared", "-o", str(LIB), *map(str, objs)]
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"link failed:\n{p.stdout}\n{p.stderr}")
    _build_bind(nvcc, force)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
