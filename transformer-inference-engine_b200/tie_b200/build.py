"""Builds libtie_b200.so in-tree with nvcc for sm_100a (no JIT cache, no torch
extension machinery): every .cu/.cpp under csrc/ is compiled to an object in
parallel, then linked into lib/libtie_b200.so; csrc/python/ops_module.cpp becomes
tie_b200/_ops (of torch only one header is used, nothing is linked).  Rebuilds only
what changed.

    python -m tie_b200.build            (from transformer-inference-engine_b200/)
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
import warnings
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
OPS_STAMP = os.path.join(OBJ_DIR, "ops_module.torch")    # the torch that it was built for

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
    """tie_b200/_ops, the Python side of the operators' calls. The library and the model do without it, so where it
    cannot be built (no torch, one without the interface that it reads tensors by, no compiler, no Python headers)
    the answer is "", with a warning unless torch is absent, and tie_b200.ops refuses its calls."""
    torch = importlib.util.find_spec("torch")
    if torch is None:
        return ""
    torch_dir = torch.submodule_search_locations[0]
    try:
        built_for = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        built_for = torch_dir
    newest = max([os.path.getmtime(OPS_SRC)] + [os.path.getmtime(os.path.join(INCLUDE, f)) for f in os.listdir(INCLUDE)])
    if os.path.exists(OPS_PATH):
        if os.path.getmtime(OPS_PATH) >= newest and _read(OPS_STAMP) == built_for:
            return OPS_PATH
        os.remove(OPS_PATH)     # it must not be called with what has changed
    os.makedirs(os.path.dirname(OPS_STAMP), exist_ok=True)
    tmp = OPS_PATH + ".tmp"
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-I" + INCLUDE,
           "-I" + sysconfig.get_paths()["include"], "-isystem", os.path.join(torch_dir, "include"), OPS_SRC, "-o", tmp]
    try:
        p = subprocess.run(cmd, capture_output=True, text=True)
        failed = p.stdout + p.stderr if p.returncode else ""
    except OSError as e:
        failed = str(e)
    if failed or not os.path.exists(tmp):
        warnings.warn(f"tie_b200._ops is not built, tie_b200.ops will not work:\n{failed[:2000]}", RuntimeWarning)
        return ""
    os.replace(tmp, OPS_PATH)
    with open(OPS_STAMP, "w") as f:
        f.write(built_for)
    return OPS_PATH


def _read(path: str) -> str:
    try:
        with open(path) as f:
            return f.read()
    except OSError:
        return ""


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
