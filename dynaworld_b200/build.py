"""Builds libgsb200.so (sm_100a) in-tree with nvcc.

    python -m dynaworld_b200.build [--verbose]

The library has no torch dependency: plain CUDA runtime (static), C ABI declared in
include/gsb200.h.  Output: dynaworld_b200/libgsb200.so, and beside it _token_torch.so, the torch
binding of the token-side operators (host code around the same C ABI).
"""
from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libgsb200.so"
SOURCES = ["abi.cu", "preprocess.cu", "sort.cu", "bin.cu", "raster.cu", "loss.cu", "splat2d.cu",
           "norm.cu", "norm_ring.cu", "linear.cu", "linear_few.cu", "linear_mma.cu", "linear_mma_bf16.cu",
           "linear_mma_f16.cu", "linear_mma_sums.cu",
           "linear_mma_f32.cu", "linear_mma_e4m3.cu"]
TORCH_SOURCE = "token_torch.cpp"  # the token-side operators' torch binding (host code, no CUDA compiler)
TORCH_LIB = PKG / "_token_torch.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; set NVCC or put the CUDA toolkit on PATH")


def needs_build() -> bool:
    if not LIB.exists() or not TORCH_LIB.exists():
        return True
    mtime = min(LIB.stat().st_mtime, TORCH_LIB.stat().st_mtime)
    deps = [CSRC / s for s in (*SOURCES, TORCH_SOURCE)] + list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list(INCLUDE.glob("*.h"))
    return any(p.stat().st_mtime > mtime for p in deps)


def torch_command(out: Path) -> list[str]:
    """g++ on the torch binding.  torch's own libraries are found at import, when torch has loaded them."""
    import sysconfig

    from torch.utils import cpp_extension

    cuda = Path(nvcc_path()).resolve().parents[1] / "include"
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], str(cuda)]
    return [shutil.which("g++") or "g++", "-O2", "-fPIC", "-shared", "-std=c++17", "-fvisibility=hidden", f"-I{INCLUDE}",
            *(a for p in include for a in ("-isystem", p)), str(CSRC / TORCH_SOURCE), "-o", str(out),
            *(f"-L{p}" for p in cpp_extension.library_paths()), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
            "-ltorch_cuda", "-ltorch_python"]


def build(force: bool = False, verbose: bool = False, ptxas_info: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    nvcc = nvcc_path()
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    common = [nvcc, *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-fvisibility=hidden",
              f"-I{INCLUDE}", f"-I{CSRC}", "--expt-relaxed-constexpr"]
    if ptxas_info:
        common.append("-Xptxas=-v")
    objs = [str(objdir / (Path(src).stem + ".o")) for src in SOURCES]
    cmds = [common + ["-c", str(CSRC / src), "-o", obj] for src, obj in zip(SOURCES, objs)]
    torch_tmp = TORCH_LIB.with_suffix(".so.tmp")
    cmds.append(torch_command(torch_tmp))
    if verbose:
        for cmd in cmds:
            print(" ".join(cmd), flush=True)
    # one compiler per source file, all at once
    procs = [subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True) for cmd in cmds]
    failed = []
    for src, proc in zip((*SOURCES, TORCH_SOURCE), procs):
        _out, err = proc.communicate()
        if proc.returncode != 0 or (verbose and err):
            sys.stderr.write(err)
        if proc.returncode != 0:
            failed.append(src)
    if failed:
        raise RuntimeError(f"the compiler failed on {', '.join(failed)}")
    os.replace(torch_tmp, TORCH_LIB)
    tmp = LIB.with_suffix(".so.tmp")
    link = [nvcc, *ARCH, "-shared", "-o", str(tmp), *objs, "-cudart", "static"]
    if verbose:
        print(" ".join(link), flush=True)
    res = subprocess.run(link, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stderr)
        raise RuntimeError("nvcc link failed")
    os.replace(tmp, LIB)
    return LIB


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    args = ap.parse_args()
    path = build(force=args.force, verbose=args.verbose, ptxas_info=args.ptxas_info)
    print(path)


if __name__ == "__main__":
    main()
