"""Builds libtie_b200.so in-tree with nvcc for sm_100a (no JIT cache, no torch
extension machinery): every .cu/.cpp under csrc/ is compiled to an object in
parallel, then linked into lib/libtie_b200.so; csrc/python/ops_module.cpp becomes
tie_b200/_ops (of torch only one header is used, nothing is linked).  Rebuilds only
what changed.

    python -m tie_b200.build            (from transformer-inference-engine_b200/)
"""
from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
REPO_ROOT = os.path.dirname(PKG_ROOT)
CSRC = os.path.join(PKG_ROOT, "csrc")
INCLUDE = os.path.join(REPO_ROOT, "include")
OBJ_DIR = os.path.join(PKG_ROOT, "build")
LIB_DIR = os.path.join(PKG_ROOT, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libtie_b200.so")

OPS_SRC = os.path.join(CSRC, "python", "ops_module.cpp")
OPS_PATH = os.path.join(PKG_ROOT, "tie_b200", "_ops" + sysconfig.get_config_var("EXT_SUFFIX"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O3",
                     "--expt-relaxed-constexpr", "-I" + INCLUDE, "-I" + CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise FileNotFoundError("nvcc not found")


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cu", ".cpp")))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def build(verbose: bool = False, extra_flags: list[str] | None = None) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    cc = nvcc()
    hdr_mtime = max(os.path.getmtime(h) for h in _headers())
    flags = NVCC_FLAGS + (extra_flags or [])

    def compile_one(src):
        obj = os.path.join(OBJ_DIR, os.path.basename(src) + ".o")
        if os.path.exists(obj) and os.path.getmtime(obj) >= max(os.path.getmtime(src), hdr_mtime):
            return obj, False
        cmd = [cc] + flags + ["-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{p.stdout}\n{p.stderr}")
        if verbose and p.stderr.strip():
            print(p.stderr, flush=True)
        return obj, True

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 2)) as ex:
        results = list(ex.map(compile_one, _sources()))
    objs = [r[0] for r in results]
    if any(r[1] for r in results) or not os.path.exists(LIB_PATH) or \
            os.path.getmtime(LIB_PATH) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB_PATH + ".tmp"
        cmd = [cc] + ARCH + ["-shared", "-o", tmp] + objs + ["-lcuda"]
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"link failed:\n{p.stdout}\n{p.stderr}")
        os.replace(tmp, LIB_PATH)
    build_ops_module()
    return LIB_PATH


def build_ops_module() -> str:
    """tie_b200/_ops, the Python side of the operators' calls ("" without torch, whose tensors it reads)."""
    torch = importlib.util.find_spec("torch")
    if torch is None:
        return ""
    newest = max([os.path.getmtime(OPS_SRC)] + [os.path.getmtime(os.path.join(INCLUDE, f)) for f in os.listdir(INCLUDE)])
    if os.path.exists(OPS_PATH) and os.path.getmtime(OPS_PATH) >= newest:
        return OPS_PATH
    torch_dir = torch.submodule_search_locations[0]
    tmp = OPS_PATH + ".tmp"
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I" + INCLUDE,
           "-I" + sysconfig.get_paths()["include"], "-isystem", os.path.join(torch_dir, "include"), OPS_SRC, "-o", tmp]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"g++ failed on {OPS_SRC}:\n{p.stdout}\n{p.stderr}")
    os.replace(tmp, OPS_PATH)
    return OPS_PATH


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
