"""Build libvcattn.so in-tree with nvcc for sm_100a.

    python -m comfyui_vc_attention_b200.build [--force] [--jobs N]

Each ``csrc/*.cu`` compiles to an object under ``_build/`` (in parallel) and
the objects link into ``comfyui_vc_attention_b200/libvcattn.so``.  The library
exports only the C ABI of ``include/vcattn.h``; it does not link against torch.
The host side of the block operators (``csrc/host_ops.cpp``) is a Python
extension over torch's tensors, ``vc_attention/_host_ops.so``, that calls that
ABI; without torch only the library is built.  A source is recompiled when it,
or any header, is newer than its object, the extension also when torch, Python
or the command changes.
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import glob
import os
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
INCLUDE = os.path.join(REPO, "include")
BUILD = os.path.join(REPO, "_build")
LIB = os.path.join(PKG, "libvcattn.so")
HOST_OPS = os.path.join(PKG, "vc_attention", "_host_ops.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "--expt-relaxed-constexpr",
              "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden",
              "-I", INCLUDE, "-I", CSRC]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found")


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.cuh")) + glob.glob(os.path.join(INCLUDE, "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _compile(src: str, obj: str, extra) -> str:
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, *extra, "-c", src, "-o", obj]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {os.path.basename(src)}:\n{r.stderr}\n{r.stdout}")
    return r.stderr


def _host_ops(force: bool) -> None:
    try:
        import torch
    except ImportError as e:
        print(f"torch cannot be imported ({e}): {os.path.basename(HOST_OPS)}, the host side of the block operators, "
              f"is not built", file=sys.stderr)
        return
    import sysconfig

    src = os.path.join(CSRC, "host_ops.cpp")
    root = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    inc = [INCLUDE, os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
           os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_host_ops",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *[f"-I{p}" for p in inc], src,
           "-o", HOST_OPS + ".tmp", "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    # what the extension was built with and for
    made = "\n".join([torch.__version__, sys.version, *cmd])
    stamp = os.path.join(BUILD, "host_ops.txt")
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(INCLUDE, "vcattn.h")))
    if not force and os.path.exists(HOST_OPS) and os.path.getmtime(HOST_OPS) >= newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == made:
                return
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for host_ops.cpp:\n{r.stderr}\n{r.stdout}")
    os.replace(HOST_OPS + ".tmp", HOST_OPS)
    with open(stamp, "w") as f:
        f.write(made)


def build(force: bool = False, jobs: int = 0, verbose: bool = False, extra=()) -> str:
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr = _headers_mtime()
    todo = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if force or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr):
            todo.append((s, o))
    jobs = jobs or min(len(todo) + 1, os.cpu_count() or 4)
    with cf.ThreadPoolExecutor(max_workers=jobs) as ex:
        host = ex.submit(_host_ops, force)
        if todo:
            futs = {ex.submit(_compile, s, o, list(extra)): s for s, o in todo}
            for f in cf.as_completed(futs):
                msg = f.result()
                if verbose and msg.strip():
                    print(f"[{os.path.basename(futs[f])}]\n{msg}", file=sys.stderr)
    if todo or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(map(os.path.getmtime, objs), default=0.0):
        cmd = [nvcc(), *ARCH, "-shared", "-Xcompiler", "-fPIC", *objs, "-o", LIB + ".tmp"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}\n{r.stdout}")
        os.replace(LIB + ".tmp", LIB)
    host.result()   # (after the link: the library does not depend on it)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=0)
    ap.add_argument("--verbose", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true", help="print registers/spills per kernel")
    args = ap.parse_args()
    extra = ["-Xptxas", "-v"] if args.ptxas_info else []
    print(build(force=args.force or args.ptxas_info, jobs=args.jobs,
                verbose=args.verbose or args.ptxas_info, extra=extra))
    return 0


if __name__ == "__main__":
    sys.exit(main())
