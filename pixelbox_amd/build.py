"""Build the HIP shared library in-tree: pixelbox_amd/libpixelbox_hip.so (gfx950 only).

hipcc cross-compiles without a GPU.  -ffp-contract=off: the exact re-scoring kernels and the host-side
query fold must round every multiply and add separately, like the reference's Rust f32 code
(engine.rs:572-588) -- the top-k order depends on it.

The gate is a CONTENT hash, not an mtime: `libpixelbox_hip.so.stamp` records the sha256 of every source,
header and the compile flags the library was built from; build() recompiles whenever the tree's hash differs
and always prints which of the two happened, so a log reader can tell whether the shipped binary is the
source's.  The translation units compile in parallel.
"""
from __future__ import annotations

import hashlib
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libpixelbox_hip.so")
STAMP = LIB + ".stamp"
SOURCES = ["pb_scan.hip", "pb_embed.hip", "pb_gemm_p3.hip", "pb_sharded.hip", "pb_phash.hip", "pb_linear.hip"]
HEADERS = ["pb_common.h", "pb_scan_kernels.h", "pb_embed_common.h", "pb_embed_kernels.h", "pb_gemm_p3.h", "pb_p3_common.h", "pb_gemm_p3_launch.h", "pb_front_band.h", "pb_block_small.h", "pb_phash_kernels.h", "pb_merge_kernels.h", "pb_linear_kernels.h",
           os.path.join("..", "..", "include", "pixelbox_hip.h")]
# no packed f32 arithmetic (v_pk_add / mul / fma_f32): some of its forms have given wrong results on this chip now and then (the
# host pass of hipcc warns that it does not know the feature: harmless)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-fno-fast-math", "-Wall",
         "-Wno-unused-function", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
# the short way from torch tensors to the linear layers' entry points (pixelbox_amd/linear.py): host code, against torch's headers
CALL_SRC = "pb_linear_call.cpp"
CALL_LIB = os.path.join(HERE, "_linear_call.so")
CALL_STAMP = CALL_LIB + ".stamp"
# RCCL (the sharded index's all-gather, pb_sharded.hip) is dlopen'ed at pb_sharded_create: a single-GPU host never loads it
LINK = ["-ldl"]


def _hipcc() -> str:
    for c in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found (need ROCm with gfx950 support)")


def _extra() -> list[str]:
    return os.environ.get("PB_EXTRA_HIPCC_FLAGS", "").split()  # kernel experiments (-D...), empty by default


def source_hash() -> str:
    h = hashlib.sha256()
    h.update(" ".join(FLAGS + _extra() + LINK).encode())
    for rel in SOURCES + HEADERS:
        p = os.path.join(CSRC, rel)
        if os.path.exists(p):
            h.update(rel.encode())
            with open(p, "rb") as f:
                h.update(f.read())
    return h.hexdigest()


def _torch_dir() -> str | None:
    spec = importlib.util.find_spec("torch")
    return os.path.dirname(spec.origin) if spec and spec.origin else None


def _stamp(path: str) -> str:
    if not os.path.exists(path):
        return ""
    with open(path) as f:
        return f.read().strip()


def _needs_lib() -> bool:
    return not os.path.exists(LIB) or _stamp(STAMP) != source_hash()


def _needs_call() -> bool:
    """whether _linear_call.so is to be tried: not where it was tried with the same sources and could not be built"""
    want = call_hash()
    return bool(want) and not (_stamp(CALL_STAMP) == want and os.path.exists(CALL_LIB)) and _stamp(CALL_STAMP) != "failed " + want


def needs_build() -> bool:
    return _needs_lib() or _needs_call()


def _compile(src: str, verbose: bool) -> str:
    obj = os.path.splitext(src)[0] + ".o"
    cmd = [_hipcc()] + _extra() + FLAGS + ["-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.check_call(cmd)
    return obj


def call_tag() -> str:
    """the torch and the Python whose layouts _linear_call.so has compiled in"""
    t, version = _torch_dir(), ""
    if t is not None:
        with open(os.path.join(t, "version.py")) as f:
            found = re.search(r"^__version__\s*=\s*['\"]([^'\"]+)", f.read(), re.M)
        version = found.group(1) if found else "unknown"
    return f"torch {version} {sysconfig.get_config_var('SOABI')}"


def _call_command() -> list[str]:
    """what compiles _linear_call.so; empty where there is no torch to build it against (a host without Python has no use for it)"""
    t = _torch_dir()
    if t is None:
        return []
    hipcc = shutil.which("hipcc")
    rocm = os.environ.get("ROCM_PATH") or (os.path.dirname(os.path.dirname(os.path.realpath(hipcc))) if hipcc else "/opt/rocm")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", f'-DPB_BUILT_FOR="{call_tag()}"',
            "-I" + os.path.join(t, "include"),
            "-I" + os.path.join(t, "include", "torch", "csrc", "api", "include"), "-I" + os.path.join(rocm, "include"), "-I" + sysconfig.get_paths()["include"],
            os.path.join(CSRC, CALL_SRC), "-o", CALL_LIB, "-L" + os.path.join(t, "lib"), "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip",
            "-Wl,-rpath," + os.path.join(t, "lib")]


def call_hash() -> str:
    cmd = _call_command()
    if not cmd:
        return ""
    h = hashlib.sha256(" ".join(cmd).encode())
    for rel in (CALL_SRC, os.path.join("..", "..", "include", "pixelbox_hip.h")):
        with open(os.path.join(CSRC, rel), "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def _build_call(verbose: bool) -> bool:
    """_linear_call.so.  It only shortens calls that pixelbox_amd/linear.py makes without it too: where it cannot be built (no headers, another
    compiler, a torch without HIP) that is said, an older one is taken away, and the library is built all the same."""
    cmd, want = _call_command(), call_hash()
    if not cmd:
        return False
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    try:
        subprocess.check_call(cmd)
    except (OSError, subprocess.CalledProcessError) as e:
        print(f"pixelbox_amd.build: {os.path.basename(CALL_LIB)} could not be built ({e}); calls from torch take the longer way", file=sys.stderr)
        if os.path.exists(CALL_LIB):
            os.remove(CALL_LIB)
        want = "failed " + want
    with open(CALL_STAMP, "w") as f:
        f.write(want + "\n")
    return not want.startswith("failed")


def _build_lib(verbose: bool) -> int:
    srcs = [os.path.join(CSRC, s) for s in SOURCES if os.path.exists(os.path.join(CSRC, s))]
    want = source_hash()
    with ThreadPoolExecutor(max_workers=min(5, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    cmd = [_hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs + LINK
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.check_call(cmd)
    with open(STAMP, "w") as f:
        f.write(want + "\n")
    return len(srcs)


def build(force: bool = False, verbose: bool = False) -> str:
    lib, call = force or _needs_lib(), force or _needs_call()
    with ThreadPoolExecutor(max_workers=1) as ex:  # beside the library's translation units
        beside = ex.submit(_build_call, verbose) if call else None
        n = _build_lib(verbose) if lib else 0
        has_call = beside.result() if beside else os.path.exists(CALL_LIB)
    if not lib and not call:
        print(f"pixelbox_amd.build: {os.path.basename(LIB)} is up to date with the sources (sha256 {_stamp(STAMP)[:16]})", file=sys.stderr)
    else:
        print(f"pixelbox_amd.build: compiled {n} translation units for gfx950 -> {os.path.basename(LIB)} "
              f"{'and _linear_call.so ' if has_call else ''}(sha256 of sources + flags {_stamp(STAMP)[:16]})", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    print(build(force="--if-needed" not in sys.argv, verbose=True))
