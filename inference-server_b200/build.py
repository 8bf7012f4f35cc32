"""Builds libb200decode.so (the C-ABI library) in-tree with nvcc for sm_100a.

Run as a script (``python inference-server_b200/build.py``) or call
:func:`build_library`.  Only what is older than its source is compiled
again.  nvcc cross-compiles without a GPU present.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
INCLUDE = os.path.join(ROOT_DIR, "include")
LIB_PATH = os.path.join(PKG_DIR, "libb200decode.so")
SOURCES = ["host.cu", "paged_attn.cu", "paged_prefill.cu", "paged_prefill_tc.cu", "paged_prefill_pairs.cu", "decode_glue.cu", "dense_gemm.cu", "router_fused.cu", "moe_route.cu", "moe_gemm.cu",
           "moe_layer.cu", "ep_p2p.cu", "latent_attn.cu", "layer_glue.cu", "gated_glue.cu", "state_scan.cu", "mixed_attn.cu",
           "mixed_prefill_tc.cu", "state_step.cu", "state_chunk.cu", "kv8_append.cu", "kv8_decode.cu", "kv8_prefill.cu"]
# Parts of the library that are enough for some model families, each with a library file of its own, for a process that
# has to build before it can run and needs no more than that.
SUBSETS = {
    "layered": ["host.cu", "paged_attn.cu", "paged_prefill.cu", "paged_prefill_tc.cu", "paged_prefill_pairs.cu", "dense_gemm.cu", "latent_attn.cu",
                "layer_glue.cu"],
    "gated": ["host.cu", "dense_gemm.cu", "moe_route.cu", "layer_glue.cu", "gated_glue.cu", "state_scan.cu", "mixed_attn.cu",
              "mixed_prefill_tc.cu", "state_step.cu", "state_chunk.cu"],
}
HEADERS = ["common.cuh", "glue.cuh", "host.h", "kv8.cuh", "prefill_tc.cuh"]
BINDING = "kv8_bind.cpp"  # a Python extension module over the C ABI (see there)
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-Xcompiler", "-fPIC", "-I", INCLUDE, "-I", CSRC,
]


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; cannot build libb200decode.so")
    return exe


def _mtime(path: str) -> float:
    return os.path.getmtime(path) if os.path.exists(path) else 0.0


def _header_time() -> float:
    return max(_mtime(os.path.join(CSRC, h)) for h in HEADERS) if HEADERS else 0.0


def _newest(sources: list[str]) -> float:
    return max([_mtime(os.path.join(CSRC, f)) for f in sources]
               + [_header_time(), _mtime(os.path.join(INCLUDE, "b200_decode.h"))])


def _fresh(path: str, sources: list[str]) -> bool:
    return _mtime(path) >= _newest(sources)


def subset_path(subset: str) -> str:
    return LIB_PATH.replace(".so", f"_{subset}.so")


def binding_path() -> str:
    """File of the native binding for the running Python and the installed torch, whose C++ classes it is compiled against: after an upgrade
    of either it is another file, which is not there yet."""
    import torch
    return os.path.join(PKG_DIR, f"_kv8-{sys.implementation.cache_tag}-torch{torch.__version__}-abi{int(torch._C._GLIBCXX_USE_CXX11_ABI)}.so")


def build_binding(force: bool = False) -> str:
    """Compile the native binding against the installed torch and Python.  Returns its path."""
    source, path = os.path.join(CSRC, BINDING), binding_path()
    if not force and _mtime(path) >= max(_mtime(source), _mtime(os.path.join(INCLUDE, "b200_decode.h"))):
        return path
    import sysconfig

    import torch
    base = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    lib = os.path.join(base, "lib")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-o", path + ".tmp", source, "-I", INCLUDE, "-I", os.path.join(base, "include"),
           "-I", os.path.join(base, "include", "torch", "csrc", "api", "include"), "-I", sysconfig.get_path("include"),
           "-I", os.path.join(cuda, "include"), f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-L", lib, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda"]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed on {BINDING}:\n{res.stdout}")
    os.replace(path + ".tmp", path)
    return path


def build_library(force: bool = False, verbose: bool = False, subset: str | None = None) -> str:
    """Compile what is out of date of the .cu files under csrc/ (of one of SUBSETS if given) and link the shared library; without a
    subset the native binding too, behind it, for the library does not need torch.  Returns the library's path."""
    sources, lib_path = (SOURCES, LIB_PATH) if subset is None else (SUBSETS[subset], subset_path(subset))
    if force or not _fresh(lib_path, sources):
        _compile_and_link(sources, lib_path, force, verbose)
    if subset is None:
        build_binding(force)
    return lib_path


def _compile_and_link(sources: list[str], lib_path: str, force: bool, verbose: bool) -> None:
    nvcc = _nvcc()
    obj_dir = os.path.join(ROOT_DIR, "build")
    os.makedirs(obj_dir, exist_ok=True)
    objs = []
    procs = []
    for src in sources:
        obj = os.path.join(obj_dir, src.replace(".cu", ".o"))
        objs.append(obj)
        if not force and _fresh(obj, [src]):
            continue
        cmd = [nvcc, *NVCC_FLAGS, "-c", os.path.join(CSRC, src), "-o", obj + ".tmp.o"]
        if verbose:
            cmd.insert(1, "-Xptxas")
            cmd.insert(2, "-v")
        procs.append((src, obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for src, obj, proc in procs:
        out, _ = proc.communicate()
        if verbose and out:
            print(out)
        if proc.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{out}")
        os.replace(obj + ".tmp.o", obj)
    tmp = lib_path + ".tmp"
    link = [nvcc, "-shared", "-o", tmp, *objs, "-gencode", "arch=compute_100a,code=sm_100a"]
    res = subprocess.run(link, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}")
    os.replace(tmp, lib_path)


def library_for(subset: str) -> str:
    """Path of an up-to-date library with the entry points of `subset`: the full one if it is there, else the subset's,
    built now if need be."""
    if _fresh(LIB_PATH, SOURCES):
        return LIB_PATH
    return build_library(subset=subset)


if __name__ == "__main__":
    path = build_library(force="--force" in sys.argv, verbose="-v" in sys.argv)
    print(path)
