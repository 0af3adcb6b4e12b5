"""Build libgdpa_b200.so (the C-ABI kernel library) in-tree with nvcc for sm_100a, and libgdpa_b200_torch.so (torch operators that
call it from C++) with the host compiler.

    python -m ads_model_kernel_library_b200.build [--force] [--verbose]

Each translation unit under csrc/ is compiled to an object file in csrc/build/ (in parallel) and
linked into ads_model_kernel_library_b200/libgdpa_b200.so.  Objects are rebuilt only when a source
or header is newer.  nvcc cross-compiles without a GPU.
"""
from __future__ import annotations

import argparse
import concurrent.futures
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
OUT = os.path.join(PKG, "libgdpa_b200.so")
TORCH_SRCS = [os.path.join(CSRC, f) for f in ("gdpa_torch.cpp", "gdpa_torch_heads.cpp")]
TORCH_OUT = os.path.join(PKG, "libgdpa_b200_torch.so")
TORCH_STAMP = os.path.join(CSRC, "build", "gdpa_torch.stamp")  # which torch it was built for
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17", "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; libgdpa_b200.so cannot be built")
    return exe


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _newest_header() -> float:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hdrs.append(os.path.join(os.path.dirname(PKG), "include", "gdpa_b200.h"))
    return max(os.path.getmtime(h) for h in hdrs)


def _build_torch_ops(force: bool, verbose: bool) -> None:
    """The torch operators, for the torch that is installed: again when it is another one than at the last build.  Without torch or g++ they are left
    out (the kernel library needs neither; the operators' first call says that they are missing)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or shutil.which("g++") is None:
        sys.stderr.write(f"{'torch' if spec is None else 'g++'} is not there: {os.path.basename(TORCH_OUT)} is not built\n")
        return
    torch = os.path.dirname(spec.origin)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    built_for = f"torch {importlib.metadata.version('torch')} in {torch}\n"
    read = [*TORCH_SRCS, os.path.join(CSRC, "gdpa_torch.h"), os.path.join(os.path.dirname(PKG), "include", "gdpa_b200.h")]
    if not force and os.path.exists(TORCH_OUT) and os.path.getmtime(TORCH_OUT) >= max(os.path.getmtime(f) for f in read):
        if os.path.exists(TORCH_STAMP):
            with open(TORCH_STAMP) as f:
                if f.read() == built_for:
                    return
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", f"-I{torch}/include", f"-I{torch}/include/torch/csrc/api/include",
           f"-I{cuda}/include", *TORCH_SRCS,
           "-o", TORCH_OUT, f"-L{torch}/lib", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError("g++ failed; see output above")
    os.makedirs(os.path.dirname(TORCH_STAMP), exist_ok=True)
    with open(TORCH_STAMP, "w") as f:
        f.write(built_for)


def build(force: bool = False, verbose: bool = False) -> str:
    nvcc = _nvcc()
    objdir = os.path.join(CSRC, "build")
    os.makedirs(objdir, exist_ok=True)
    hdr_time = _newest_header()
    jobs, objs = [], []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_time):
            cmd = [nvcc, *NVCC_FLAGS, "-c", s, "-o", o]
            if verbose:
                cmd.insert(1, "-Xptxas=-v")
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    failed = False
    with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as ex:
        for cmd, r in ex.map(run, jobs):
            if verbose or r.returncode != 0:
                sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
            failed |= r.returncode != 0
    if failed:
        raise RuntimeError("nvcc failed; see output above")
    if jobs or force or not os.path.exists(OUT):
        cmd = [nvcc, "-shared", "-o", OUT, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link of libgdpa_b200.so failed")
    _build_torch_ops(force, verbose)
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
