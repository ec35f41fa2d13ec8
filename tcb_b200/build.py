"""Build libtcb.so (the sm_100a kernels + C ABI) in-tree with nvcc, and
_tcb_torch.so (its serving entry points for torch tensors) with g++.

    python -m tcb_b200.build          # or tcb_b200.build.build()

The libraries land next to this file (tcb_b200/libtcb.so, _tcb_torch.so) so they
travel with the source tree; nothing is installed into site-packages.  libtcb.so
needs nvcc alone: without torch it is built and _tcb_torch.so is left out.
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtcb.so")
TORCH_LIB = os.path.join(HERE, "_tcb_torch.so")
CXX = os.environ.get("CXX", "g++")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]
SOURCES = ["tcb_capi.cu", "tcb_dequant.cu", "tcb_gemv_simt.cu", "tcb_matvec.cu", "tcb_mv_q4k.cu", "tcb_mv_q6k.cu", "tcb_gemm_tc.cu", "tcb_gemm_i8.cu", "tcb_mv_rows.cu", "tcb_llama.cu", "tcb_static.cu", "tcb_attn_prefill.cu",
           "tcb_serve.cu", "tcb_page_decode.cu", "tcb_page_rows.cu", "tcb_logits.cu"]


def _stale(objs, deps) -> bool:
    if not all(os.path.exists(o) for o in objs):
        return True
    newest = max(os.path.getmtime(d) for d in deps)
    return any(os.path.getmtime(o) < newest for o in objs)


def _torch_command():
    """The compiler's command for _tcb_torch.so; None without torch."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    t = list(spec.submodule_search_locations)[0]
    return [CXX, "-O2", "-std=c++17", "-shared", "-fPIC", "-D_GLIBCXX_USE_CXX11_ABI=1",
            "-I" + sysconfig.get_paths()["include"], "-isystem", os.path.join(t, "include"), "-isystem",
            os.path.join(t, "include", "torch", "csrc", "api", "include"), "-isystem", "/usr/local/cuda/include",
            os.path.join(CSRC, "tcb_torch.cpp"), "-o", TORCH_LIB, "-L" + os.path.join(t, "lib"), "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch_python"]


def _torch_stamp() -> str:
    """What _tcb_torch.so was built against: the Python and torch it only works with."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        version = "?"
    return f"{sys.version} torch {version}\n"


def _read(path: str) -> str:
    if not os.path.exists(path):
        return ""
    with open(path) as f:
        return f.read()


def build(verbose: bool = False, force: bool = False) -> str:
    bdir = os.path.join(HERE, "_build")
    os.makedirs(bdir, exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    headers.append(os.path.join(os.path.dirname(HERE), "include", "tcb.h"))
    objs, cmds = [], []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(bdir, src.replace(".cu", ".o"))
        objs.append(o)
        if force or _stale([o], [s] + headers):
            cmds.append([NVCC, *ARCH, *FLAGS, "-c", s, "-o", o])

    torch_cmd, stamp = _torch_command(), os.path.join(bdir, "tcb_torch.stamp")
    if torch_cmd is None:
        print("torch is not installed: _tcb_torch.so (tcb_b200.serve) is left out", file=sys.stderr, flush=True)
    elif force or _stale([TORCH_LIB], [os.path.join(CSRC, "tcb_torch.cpp"), headers[-1]]) or _read(stamp) != _torch_stamp():
        cmds.append(torch_cmd)

    def compile_one(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    # the translation units are independent: compile them side by side
    with ThreadPoolExecutor(max_workers=max(1, min(len(cmds), os.cpu_count() or 1))) as ex:
        for f in [ex.submit(compile_one, c) for c in cmds]:
            f.result()
    if torch_cmd in cmds:
        with open(stamp, "w") as f:
            f.write(_torch_stamp())
    if force or _stale([LIB], objs):
        cmd = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return LIB


if __name__ == "__main__":
    build(verbose=True, force="--force" in sys.argv)
