"""Build libr3d_b200.so (the plugin) in-tree with nvcc for sm_100a.

    python -m libr3d_b200.build

The shared object lands next to this file so that it travels with the source tree; there
is no JIT cache and no installed copy. Building it needs nvcc alone. Where torch is installed,
_bind.so (the Python side of the int8 step) is built beside it, and again after a change of
torch. Objects are rebuilt only when a source or header is newer. `-fmad=false`: the kernels
spell every fused multiply-add they want, because a contracted mul+add is a different rounding
than the arithmetic contract states.
"""
from __future__ import annotations

import concurrent.futures as cf
import importlib.util
import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
OBJ = PKG / "build"
SO = PKG / "libr3d_b200.so"
BIND = PKG / "_bind.so"
BIND_FOR = OBJ / "bind_for.txt"                   # the torch that _bind.so was built against

SOURCES = [
    "rows_table.cpp",
    "entries_gemm_q.cpp",
    "entries_band.cpp",
    "entries_logits.cpp",
    "entries_w2a8.cpp",
    "entries_i8.cpp",
    "planes_cache.cpp",
    "launch.cu",
    "kern_exact.cu",
    "kern_topk.cu",
    "kern_rerank.cu",
    "kern_w2a8.cu",
    "kern_q8x.cu",
    "kern_i8.cu", "kern_token_i8.cu", "kern_nucleus.cu",
    "q8x_static.cu",
    "kern_stream.cu",
    "kern_tc.cu", "kern_tc_mxf4.cu", "kern_tc_q8x.cu", "kern_tc_gemm.cu", "kern_tc_gemm2.cu", "kern_tc_i8.cu", "gather.cu",
]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-lineinfo", "-O3", "-std=c++17", "-fmad=false",
    "-Xcompiler", "-fPIC,-Wall,-Wno-unused-function",
    "-I", str(ROOT / "include"), "-I", str(CSRC),
]


def _nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_plugin(verbose: bool = False, ptxas_info: bool = False) -> Path:
    OBJ.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + list((ROOT / "include").glob("*.h"))
    srcs = [s for s in SOURCES if (CSRC / s).exists()]
    jobs = []
    for s in srcs:
        src = CSRC / s
        obj = OBJ / (src.stem + ".o")
        if _stale(obj, [src] + headers):
            cmd = [_nvcc(), *NVCC_FLAGS, "-x", "cu", "-c", str(src), "-o", str(obj)]
            if ptxas_info:
                cmd[1:1] = ["-Xptxas", "-v"]
            jobs.append((s, cmd))
    if jobs:
        with cf.ThreadPoolExecutor(max_workers=min(8, len(jobs))) as ex:
            futs = {ex.submit(subprocess.run, cmd, capture_output=True, text=True): s for s, cmd in jobs}
            for f in cf.as_completed(futs):
                r = f.result()
                if verbose or r.returncode != 0 or ptxas_info:
                    sys.stderr.write(f"[{futs[f]}]\n{r.stdout}{r.stderr}\n")
                if r.returncode != 0:
                    raise RuntimeError(f"nvcc failed on {futs[f]}")
    objs = [OBJ / (Path(s).stem + ".o") for s in srcs]
    if jobs or _stale(SO, objs):
        cmd = [_nvcc(), "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(SO),
               *map(str, objs)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return SO


def build_bind() -> Path:
    """_bind.so: ops.py's call path in C++ (torch's headers, the plugin beside it)."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    src = CSRC / "bind.cpp"
    against = f"torch {torch.__version__} {sys.implementation.cache_tag}"
    if _stale(BIND, [src, SO, *(ROOT / "include").glob("*.h")]) or not BIND_FOR.exists() or BIND_FOR.read_text() != against:
        home = Path(torch.__file__).resolve().parent
        cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               *(f"-isystem{p}" for p in cpp_extension.include_paths("cuda")), f"-isystem{sysconfig.get_paths()['include']}",
               "-I", str(ROOT / "include"), str(src), "-o", str(BIND),
               f"-L{home / 'lib'}", "-ltorch_python", "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_cuda",
               f"-L{PKG}", f"-l:{SO.name}", "-Wl,-rpath,$ORIGIN"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("g++ failed on bind.cpp")
        OBJ.mkdir(exist_ok=True)
        BIND_FOR.write_text(against)
    return BIND


if __name__ == "__main__":
    build_plugin(verbose="-v" in sys.argv, ptxas_info="--ptxas" in sys.argv)
    print(SO)
    if importlib.util.find_spec("torch") is None:
        sys.stderr.write("torch is not installed: _bind.so, which ops.py's int8 step goes through, is not built\n")
    else:
        print(build_bind())
