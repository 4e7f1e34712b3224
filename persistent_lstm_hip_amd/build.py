"""Build recipe of the native library (hipcc, gfx950 only).

    python -m persistent_lstm_hip_amd.build        # -> persistent_lstm_hip_amd/lib/libpersistent_lstm_hip.so

The library exposes the C ABI declared in include/persistent_lstm_hip.h.  Beside it the module plh_torch.so, the
torch front end of the block operators, is compiled as plain C++ against the installed torch.  Both are built in-tree so
that they travel with the source tree; nothing is installed.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PKG_DIR)
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_DIR = os.path.join(PKG_DIR, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libpersistent_lstm_hip.so")
TORCH_PATH = os.path.join(LIB_DIR, "plh_torch.so")
BENCH_PATH = os.path.join(LIB_DIR, "plh_bench")
SOURCES = ["plh_wavefront.hip", "plh_sliced.hip", "plh_rec.hip", "plh_gemm.hip", "plh_pack.hip", "plh_launch.hip",
           "plh_probe.hip", "plh_capi.hip", "plh_scan.hip", "plh_norm.hip", "plh_dropout.hip",
           "plh_conv.hip", "plh_selective.hip", "plh_clip.hip"]
HEADERS = ["plh_internal.h", "plh_device.h", "plh_ops.h", os.path.join("..", "..", "include", "persistent_lstm_hip.h")]

ARCH = "gfx950"
HIPCC_FLAGS = [
    "-O3",
    "-std=c++17",
    f"--offload-arch={ARCH}",
    "-fPIC",
    # Keep packed-FP32 VALU ops out of the generated code (v_pk_{add,mul,fma}_f32).
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall",
    "-Wno-unused-command-line-argument",
]
# Only the HIP runtime (hipcc links it); every kernel is in csrc/, no vendor math library.
LINK_FLAGS: list = []


def hipcc() -> str:
    path = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(path):
        raise RuntimeError("hipcc not found: the native library needs ROCm's hipcc")
    return path


def host_compiler() -> str:
    path = shutil.which("g++") or shutil.which("c++")
    if path is None:
        raise RuntimeError("g++ not found: the torch front end needs a C++ compiler")
    return path


def build(verbose: bool = False) -> str:
    """Compile every source for gfx950 and link the shared library, its native driver and the torch front end.  Always
    recompiles.  The front end comes last: without a C++ compiler or Python's headers for it this raises, with the
    library and its driver built."""
    os.makedirs(LIB_DIR, exist_ok=True)
    tmp = LIB_PATH + ".tmp"

    def run(cmd: list) -> None:
        if verbose:
            print(" ".join(cmd), flush=True)
        proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        out = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops" not in l)
        if proc.returncode != 0:
            raise RuntimeError(f"{os.path.basename(cmd[0])} failed ({proc.returncode}):\n{out}")
        if verbose and out.strip():
            print(out, flush=True)

    def compile_one(source: str, objects: str) -> str:
        obj = os.path.join(objects, source + ".o")
        run([hipcc()] + HIPCC_FLAGS + ["-c", os.path.join(CSRC, source), "-o", obj])
        return obj

    def compile_front(obj: str) -> list:
        """Compiles the torch front end; the command that links it."""
        import torch

        torch_dir = os.path.dirname(torch.__file__)
        rocm = os.path.dirname(os.path.dirname(os.path.realpath(hipcc())))
        include = [os.path.join(torch_dir, "include"), os.path.join(torch_dir, "include", "torch", "csrc", "api", "include"),
                   os.path.join(rocm, "include"), sysconfig.get_paths()["include"]]
        run([host_compiler(), "-std=c++17", "-O2", "-fPIC", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
             "-DTORCH_EXTENSION_NAME=plh_torch"] + [a for d in include for a in ("-isystem", d)] +
            ["-c", os.path.join(CSRC, "plh_torch.cpp"), "-o", obj])
        return [host_compiler(), "-shared", obj, "-L" + os.path.join(torch_dir, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip",
                "-ltorch", "-ltorch_python", "-L" + LIB_DIR, "-lpersistent_lstm_hip", "-Wl,-rpath,$ORIGIN"]

    with tempfile.TemporaryDirectory() as objects, ThreadPoolExecutor(4) as pool:
        front = pool.submit(compile_front, os.path.join(objects, "plh_torch.o"))
        objs = list(pool.map(lambda s: compile_one(s, objects), SOURCES))
        run([hipcc(), "-shared", "-fPIC", f"--offload-arch={ARCH}"] + objs + LINK_FLAGS + ["-o", tmp])
        os.replace(tmp, LIB_PATH)
        # Native driver of the C ABI (profiling target and integration example), linked to the library.
        # (plh_issue_probe.hip: a developer probe kernel of plh_bench --issue, not part of the library.)
        run([hipcc(), "-O3", "-std=c++17", f"--offload-arch={ARCH}", "-Xclang", "-target-feature", "-Xclang",
             "-packed-fp32-ops", "-Wno-unused-command-line-argument", os.path.join(CSRC, "plh_bench_main.cpp"),
             os.path.join(CSRC, "plh_issue_probe.hip"), "-L" + LIB_DIR, "-lpersistent_lstm_hip", "-Wl,-rpath,$ORIGIN",
             "-o", BENCH_PATH + ".tmp"])
        os.replace(BENCH_PATH + ".tmp", BENCH_PATH)
        run(front.result() + ["-o", TORCH_PATH + ".tmp"])
        os.replace(TORCH_PATH + ".tmp", TORCH_PATH)
    return LIB_PATH


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
