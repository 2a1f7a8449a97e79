"""Build recipe for libsinkslot_b200.so (in-tree, sm_100a).

``python -m sinkslot_b200.build`` compiles every ``csrc/*.cu`` with nvcc for
``sm_100a`` and links them into ``sinkslot_b200/libsinkslot_b200.so`` (static
cudart, C ABI declared in ``include/sinkslot_b200.h``).  Objects go to
``sinkslot_b200/_build/``; sources are rebuilt only when they, or a header,
changed.  ``csrc/torch_ops.cpp`` (the training operators' PyTorch bindings, host
code only) becomes ``sinkslot_b200/libsinkslot_b200_torch.so``, linked to that
library and to the installed torch.
"""

from __future__ import annotations

import glob
import os
import shutil
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "libsinkslot_b200.so")
TORCH_SRC = os.path.join(CSRC, "torch_ops.cpp")
TORCH_LIB = os.path.join(HERE, "libsinkslot_b200_torch.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
    "-I" + os.path.join(ROOT, "include"),
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the sm_100a extension cannot be built")


def _headers_mtime() -> float:
    hs = glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh"))
    hs += glob.glob(os.path.join(ROOT, "include", "*.h"))
    return max((os.path.getmtime(h) for h in hs), default=0.0)


def _replace(new: str, path: str) -> None:
    """Puts a built library in its place.  What a process has loaded stays loaded."""
    os.replace(new, path)
    from . import _lib
    if _lib.opened():
        warnings.warn(f"{os.path.basename(path)} was built while an older one is loaded: it is "
                      f"used from a new process on", RuntimeWarning, stacklevel=3)


def _build_torch_ops(verbose: bool) -> None:
    """libsinkslot_b200_torch.so, when its source, the C header or torch changed."""
    import torch
    stamp = os.path.join(BUILD, "torch_version")
    header = os.path.join(ROOT, "include", "sinkslot_b200.h")
    if os.path.exists(TORCH_LIB) and os.path.exists(stamp):
        newest = max(os.path.getmtime(TORCH_SRC), os.path.getmtime(header))
        if os.path.getmtime(TORCH_LIB) >= newest and open(stamp).read() == torch.__version__:
            return
    t = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(os.path.realpath(_nvcc())))
    tmp = f"{TORCH_LIB}.{os.getpid()}.tmp"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", os.path.join(t, "include"),
           "-isystem", os.path.join(t, "include", "torch", "csrc", "api", "include"),
           "-isystem", os.path.join(cuda, "include"), TORCH_SRC, "-o", tmp,
           "-L" + HERE, "-l:" + os.path.basename(LIB), "-L" + os.path.join(t, "lib"),
           "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-Wl,-rpath,$ORIGIN"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"g++ does not run: {e}") from e
    if verbose or r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError("g++ failed for csrc/torch_ops.cpp")
    _replace(tmp, TORCH_LIB)
    with open(stamp, "w") as f:
        f.write(torch.__version__)


def build(verbose: bool = False, ptxas_info: bool = False) -> str:
    nvcc = _nvcc()
    os.makedirs(BUILD, exist_ok=True)
    srcs = sorted(glob.glob(os.path.join(CSRC, "*.cu")))
    hdr_t = _headers_mtime()
    jobs = []
    objs = []
    for s in srcs:
        o = os.path.join(BUILD, os.path.basename(s)[:-3] + ".o")
        objs.append(o)
        if ptxas_info or not os.path.exists(o) or os.path.getmtime(o) < max(os.path.getmtime(s), hdr_t):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if ptxas_info else []) + ["-c", s, "-o", o]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or ptxas_info or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed for {cmd[-3]}")
    if jobs or not os.path.exists(LIB) or os.path.getmtime(LIB) < max(os.path.getmtime(o) for o in objs):
        tmp = LIB + ".tmp"
        cmd = [nvcc] + ARCH + ["-shared", "-o", tmp] + objs + ["-Xcompiler", "-fPIC"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
            raise RuntimeError("link of libsinkslot_b200.so failed")
        _replace(tmp, LIB)
    try:
        _build_torch_ops(verbose)
    except RuntimeError as e:  # the solver does without them
        header = os.path.join(ROOT, "include", "sinkslot_b200.h")
        if os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) < max(
                os.path.getmtime(TORCH_SRC), os.path.getmtime(header)):
            os.remove(TORCH_LIB)  # its calls are another library's
        warnings.warn(f"the training operators are not built: {e}", RuntimeWarning, stacklevel=2)
    return LIB


if __name__ == "__main__":
    build(verbose="-v" in sys.argv, ptxas_info="--ptxas" in sys.argv)
    print(LIB)
    sys.exit(0 if os.path.exists(TORCH_LIB) else 1)
