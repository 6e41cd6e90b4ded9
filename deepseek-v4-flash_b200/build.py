"""Build libqcau_b200.so (all CUDA sources, sm_100a) in-tree with nvcc, and the
Python binding of its short calls (csrc/bind.cpp, against torch's headers) with g++.

    python deepseek-v4-flash_b200/build.py [--jobs N] [--verbose-ptxas] [--force]

Objects go to deepseek-v4-flash_b200/_build/, the shared library to
deepseek-v4-flash_b200/qcau_b200/libqcau_b200.so and _bind.so beside it.  A source
is recompiled when it or any header under csrc/ or include/ is newer than its object,
the binding also when torch or Python are others than it was built for.  Without torch
the library is built alone.
"""
from __future__ import annotations

import argparse
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD = PKG_DIR / "_build"
LIB = PKG_DIR / "qcau_b200" / "libqcau_b200.so"
BIND = PKG_DIR / "qcau_b200" / "_bind.so"
BIND_STAMP = BUILD / "bind.stamp"  # the torch and Python that BIND was built for
SOURCES = ["capi.cu", "act_quant.cu", "rope_norm.cu", "fp8_gemm.cu", "bmm.cu",
           "attn_combine.cu", "attn_decode_sm100.cu", "attn_gather_sm100.cu", "kv_build.cu", "indexer.cu", "compress.cu",
           "indexer_score_sm100.cu", "attn_tree_sm100.cu", "attn_weights_sm100.cu", "evict.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
         "-I", str(REPO / "include")]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _headers_mtime() -> float:
    hs = list(CSRC.glob("*.cuh")) + list(CSRC.glob("*.h")) + list((REPO / "include").glob("*.h"))
    return max((h.stat().st_mtime for h in hs), default=0.0)


def build(jobs: int = 8, verbose_ptxas: bool = False, force: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    hdr = _headers_mtime()
    cc = nvcc()
    extra = ["-Xptxas", "-v"] if verbose_ptxas else []

    def compile_one(src: str):
        s = CSRC / src
        o = BUILD / (Path(src).stem + ".o")
        if not force and o.exists() and o.stat().st_mtime >= max(s.stat().st_mtime, hdr):
            return o, ""
        cmd = [cc, *ARCH, *FLAGS, *extra, "-c", str(s), "-o", str(o)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
        return o, r.stderr

    with ThreadPoolExecutor(max_workers=jobs) as ex:
        results = list(ex.map(compile_one, SOURCES))
    for _, log in results:
        if log and verbose_ptxas:
            print(log, file=sys.stderr)
    objs = [str(o) for o, _ in results]
    if force or not LIB.exists() or LIB.stat().st_mtime < max(Path(o).stat().st_mtime for o in objs):
        cmd = [cc, *ARCH, "-shared", "-o", str(LIB), *objs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    build_bind(force)
    return LIB


def build_bind(force: bool = False) -> None:
    """_bind.so: calls libqcau_b200.so (beside it) on torch tensors.  It holds for
    one torch and one Python, which BIND_STAMP names."""
    src = CSRC / "bind.cpp"
    if importlib.util.find_spec("torch") is None:
        print("torch is not installed: the library is built without its Python binding", file=sys.stderr)
        return
    stamp = f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}\n"
    if (not force and BIND.exists() and BIND.stat().st_mtime >= max(src.stat().st_mtime, _headers_mtime())
            and BIND_STAMP.exists() and BIND_STAMP.read_text() == stamp):
        return
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-DUSE_CUDA",
           "-I", str(REPO / "include"), "-I", str(root / "include"),
           "-I", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-I", str(cuda / "include"), "-I", sysconfig.get_paths()["include"], str(src),
           "-o", str(BIND), "-L", str(root / "lib"), "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu",
           "-lc10_cuda", "-lc10", "-L", str(LIB.parent), f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"binding failed:\n{r.stdout}\n{r.stderr}")
    BIND_STAMP.parent.mkdir(parents=True, exist_ok=True)
    BIND_STAMP.write_text(stamp)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=8)
    ap.add_argument("--verbose-ptxas", action="store_true")
    ap.add_argument("--force", action="store_true")
    a = ap.parse_args()
    print(build(a.jobs, a.verbose_ptxas, a.force))
