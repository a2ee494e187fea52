"""Build libmdx.so (every HIP kernel of the package, gfx950) and _bind.so (the torch binding of the serving
step's calls: the paged cache's and verify_drafts) in-tree, next to the Python shim.

    python comfy-mono-decode-xpu_amd/build.py [--jobs N]

Each source under csrc/ is compiled to an object with hipcc in parallel, then linked into
mdx/libmdx.so. The build always recompiles (it is the "does it build" check).
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "mdx", "libmdx.so")
BIND = os.path.join(CSRC, "mdx_bind.cpp")  # host code over torch's headers: a module of its own
BIND_OUT = os.path.join(HERE, "mdx", "_bind.so")
ARCH = os.environ.get("MDX_ARCH", "gfx950")

# -ffp-contract=off: every rounding the operator contracts name is an explicit single op; the
# compiler must not fuse a product into a following sum behind our back.
# -packed-fp32-ops is disabled: packed FP32 VALU forms are not used anywhere in this library.
COMMON = ["-O3", "-fPIC", "-std=c++17", "-ffp-contract=off", f"--offload-arch={ARCH}",
          "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-command-line-argument"]


def hipcc():
    for c in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if c and os.path.exists(c):
            return c
    raise RuntimeError("hipcc not found")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".cpp")) and f != os.path.basename(BIND))


def _bind(tmp_out):
    """The torch binding, with the host compiler; torch's libraries are in the process before it loads (no run path)."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    rocm = os.path.dirname(os.path.dirname(os.path.realpath(hipcc())))
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *(x for d in (sysconfig.get_paths()["include"], f"{root}/include", f"{root}/include/torch/csrc/api/include", f"{rocm}/include")
             for x in ("-isystem", d)), BIND, "-o", tmp_out, f"-L{root}/lib",
           "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if r.stderr:
        print(r.stderr, file=sys.stderr)  # (warnings)


def _compile(cc, src, obj):
    cmd = [cc, *COMMON, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    return obj


def build(jobs: int | None = None, verbose: bool = False) -> str:
    cc = hipcc()
    srcs = sources()
    jobs = jobs or min(len(srcs), int(os.environ.get("MAX_JOBS", os.cpu_count() or 4)), 16)
    with tempfile.TemporaryDirectory(prefix="mdx_build_") as tmp:
        objs = [os.path.join(tmp, os.path.basename(s) + ".o") for s in srcs]
        with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
            bind = ex.submit(_bind, BIND_OUT + ".tmp")
            list(ex.map(lambda so: _compile(cc, *so), zip(srcs, objs)))
        tmp_out = OUT + ".tmp"
        cmd = [cc, f"--offload-arch={ARCH}", "-shared", "-fPIC", *objs, "-o", tmp_out]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        os.replace(tmp_out, OUT)
    # The library is whole without the binding, which needs a host compiler and torch's headers; without it the paged cache's
    # calls raise (mdx._lib.bind), and an older one does not stay beside a newer library.
    try:
        bind.result()
    except Exception as e:
        if os.path.exists(BIND_OUT):
            os.remove(BIND_OUT)
        raise RuntimeError(f"{OUT} is built, {os.path.basename(BIND_OUT)} is not: {e}") from e
    os.replace(BIND_OUT + ".tmp", BIND_OUT)
    if verbose:
        print(f"built {OUT} from {len(srcs)} sources, {BIND_OUT}")
    return OUT


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args()
    try:
        build(args.jobs, verbose=True)
    except RuntimeError as e:
        print(e, file=sys.stderr)
        sys.exit(1)
