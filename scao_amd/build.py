"""Build the gfx950 HIP library ``scao_amd/_lib/libscao_amd.so`` in-tree.

Every ``csrc/*.hip`` file is compiled with hipcc for gfx950 only, in
parallel, and linked into one shared object exporting the C ABI declared in
``include/scao_amd.h``.  Arithmetic contraction is off (-ffp-contract=off):
fused multiply-adds are written explicitly where the reference rounds once.
Packed fp32 instructions are disabled for all device code.

``csrc/torch_host.cpp`` is host code against torch's headers: the Python module
``scao_amd._torch_host`` (``scao_amd/_torch_host.so``), built by g++.
"""

from __future__ import annotations

import concurrent.futures as cf
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
LIB = os.path.join(OUT_DIR, "libscao_amd.so")
TORCH_HOST = os.path.join(HERE, "_torch_host.so")
ROCM = os.path.dirname(os.path.dirname(os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")))
CXX = os.environ.get("CXX", "g++")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-unused-variable",
    "-I", os.path.join(ROOT, "include"),
]


def _compile(src: str, obj: str) -> str:
    cmd = [HIPCC, *FLAGS, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"hipcc failed for {os.path.basename(src)}:\n{r.stderr}")
    noise = "is not a recognized feature for this target"
    return "\n".join(ln for ln in r.stderr.splitlines() if noise not in ln and ln.strip())


def _compile_torch_host() -> str:
    from torch._C import _GLIBCXX_USE_CXX11_ABI as abi
    from torch.utils import cpp_extension
    root = os.path.dirname(os.path.dirname(cpp_extension.__file__))
    inc = [f"-I{d}" for d in (os.path.join(root, "include"),
                              os.path.join(root, "include", "torch", "csrc", "api", "include"),
                              sysconfig.get_path("include"), os.path.join(ROCM, "include"))]
    tmp = TORCH_HOST + ".tmp"
    cmd = [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(abi)}",
           "-DUSE_ROCM", "-D__HIP_PLATFORM_AMD__", *inc, os.path.join(CSRC, "torch_host.cpp"),
           "-o", tmp, "-L" + os.path.join(root, "lib"), "-ltorch_python", "-ltorch_cpu",
           "-lc10_hip", "-lc10"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{CXX} failed for torch_host.cpp:\n{r.stderr}")
    os.replace(tmp, TORCH_HOST)
    return r.stderr


def build(verbose: bool = False) -> str:
    os.makedirs(OUT_DIR, exist_ok=True)
    srcs = sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))
    objs = [os.path.join(OUT_DIR, f[:-4] + ".o") for f in srcs]
    with cf.ThreadPoolExecutor(max_workers=8) as ex:
        torch_host = ex.submit(_compile_torch_host)
        futs = {ex.submit(_compile, os.path.join(CSRC, s), o): s for s, o in zip(srcs, objs)}
        for fut in cf.as_completed(futs):
            msg = fut.result()
            if verbose and msg:
                print(f"[{futs[fut]}]\n{msg}", file=sys.stderr)
        torch_host.result()
    tmp = LIB + ".tmp"
    cmd = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", tmp, *objs]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stderr}")
    os.replace(tmp, LIB)
    for o in objs:
        os.remove(o)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))
