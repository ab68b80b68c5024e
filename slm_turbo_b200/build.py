"""Build the sm_100a C-ABI library ``libslm_turbo_b200.so`` in-tree with nvcc,
and the Python module ``_host.so`` (host side of the serving-step entry points,
a C++ file on top of the library and torch's headers) with g++.

    python -m slm_turbo_b200.build          # or build_library() from Python

Both are written next to this file so that they travel with the source tree;
there is no JIT cache.  The library needs nvcc alone; the module, torch (with
its headers) and g++: where they are missing the library is built all the same.  Flags of the library: sm_100a
only, -O3, -lineinfo, IEEE division/rounding (no --use_fast_math: the
quantizers must match the reference bit for bit).
"""
from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
CSRC = HERE / "csrc"
INCLUDE = ROOT / "include"
LIB_NAME = "libslm_turbo_b200.so"
LIB_PATH = HERE / LIB_NAME
HOST_PATH = HERE / "_host.so"
HOST_SOURCE = CSRC / "host.cpp"
HOST_STAMP = HERE / "_build" / "host.stamp"  # what _host.so was built for
SOURCES = ["decode.cu", "store.cu", "decode_noalloc.cu",
           "decode_d64_paged.cu", "decode_d64_contig.cu", "decode_d80_paged.cu", "decode_d80_contig.cu",
           "decode_d128_paged.cu", "decode_d128_contig.cu", "prefill.cu",
           "page_ops.cu", "rotary.cu", "prompt.cu"]
HEADERS = ["ptx.cuh", "decode_common.cuh", "decode_kernels.cuh", "decode_dispatch.cuh", "quant_store.cuh",
           "internal.h", "tcgen05.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "--expt-relaxed-constexpr",
    "-Xcompiler", "-fPIC,-O3",
    "-cudart", "shared",
]


def nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def _stale() -> bool:
    if not LIB_PATH.exists():
        return True
    t = LIB_PATH.stat().st_mtime
    deps = [CSRC / s for s in SOURCES + HEADERS] + [INCLUDE / "slm_turbo_b200.h"]
    return any(d.stat().st_mtime > t for d in deps)


def _torch_root():
    """Where torch is installed (not imported), None if it is not."""
    spec = importlib.util.find_spec("torch")
    return Path(spec.origin).resolve().parent if spec and spec.origin else None


def _host_tools():
    """What _host.so is built with: (paths by name, None), or (None, what is missing)."""
    root, toolkit = _torch_root(), shutil.which(nvcc())
    # the system's g++ and not $CXX: the module throws and formats through the
    # libstdc++ that torch has loaded, and a compiler that links its own copy
    # in makes one that crashes
    paths = {"torch": root, "cxx": shutil.which("g++"), "python": Path(sysconfig.get_paths()["include"]),
             "cuda": Path(toolkit).resolve().parent.parent / "include" if toolkit else None}
    missing = ("torch" if root is None else
               "torch's CUDA headers and libraries" if not ((root / "include/ATen/cuda/EmptyTensor.h").exists()
                                                            and (root / "lib/libc10_cuda.so").exists()) else
               "g++" if paths["cxx"] is None else
               "Python.h" if not (paths["python"] / "Python.h").exists() else
               "the CUDA headers" if not (toolkit and (paths["cuda"] / "cuda_runtime_api.h").exists()) else None)
    return (None, missing) if missing else (paths, None)


def _host_built_for() -> str:
    """The torch and the Python that a module built now belongs to."""
    try:
        torch_version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        torch_version = "unknown"
    return f"torch {torch_version}, {sysconfig.get_config_var('SOABI')}\n"


def build_host(force: bool = False, verbose: bool = False):
    """Compile the Python module on top of the library (skips if it is up to
    date, and built for this torch and Python).  Where torch or a C++ toolchain
    is missing it says so and returns None: the library does not need them."""
    tools, missing = _host_tools()
    if missing:
        print(f"_host.so is not built: {missing} not found (the C library does not need it; the serving-step "
              "functions in Python do)", file=sys.stderr)
        return None
    built_for = _host_built_for()
    deps = [HOST_SOURCE, INCLUDE / "slm_turbo_b200.h"]
    if (not force and HOST_PATH.exists() and all(d.stat().st_mtime <= HOST_PATH.stat().st_mtime for d in deps)
            and HOST_STAMP.exists() and HOST_STAMP.read_text() == built_for):
        return HOST_PATH
    import torch
    root = tools["torch"]
    tmp = HOST_PATH.with_suffix(".so.tmp")
    cmd = [tools["cxx"], "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-I", str(INCLUDE),
           "-I", str(tools["cuda"]), "-isystem", str(root / "include"),
           "-isystem", str(root / "include/torch/csrc/api/include"), "-I", str(tools["python"]),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", str(HOST_SOURCE), "-o", str(tmp),
           "-L", str(LIB_PATH.parent), f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN",
           "-L", str(root / "lib"), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, HOST_PATH)
    HOST_STAMP.parent.mkdir(exist_ok=True)
    HOST_STAMP.write_text(built_for)
    return HOST_PATH


def build_library(force: bool = False, verbose: bool = False, extra_flags=None) -> Path:
    """Compile every .cu source into one shared library (skips if up to date)."""
    if not force and not _stale():
        build_host(verbose=verbose)
        return LIB_PATH
    build_dir = HERE / "_build"
    build_dir.mkdir(exist_ok=True)
    flags = NVCC_FLAGS + list(extra_flags or [])
    cmds = []
    for src in SOURCES:
        obj = build_dir / (Path(src).stem + ".o")
        cmds.append(([nvcc(), *flags, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(CSRC / src), "-o", str(obj)],
                     str(obj)))

    def compile_one(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        return subprocess.run(cmd, capture_output=not verbose, text=True)

    # the translation units are independent: compile them in parallel
    with ThreadPoolExecutor(max_workers=min(len(cmds), os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, [c for c, _ in cmds]))
    for (cmd, _), res in zip(cmds, results):
        if res.returncode != 0:
            sys.stderr.write((res.stdout or "") + (res.stderr or ""))
            raise subprocess.CalledProcessError(res.returncode, cmd, res.stdout, res.stderr)
        if not verbose and extra_flags and res.stderr:
            sys.stderr.write(res.stderr)
    objs = [o for _, o in cmds]
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-cudart", "shared",
           "-Xlinker", "-rpath,/usr/local/cuda/lib64", *objs, "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB_PATH)
    build_host(force=force, verbose=verbose)
    return LIB_PATH


if __name__ == "__main__":
    force = "--force" in sys.argv
    extra = ["-Xptxas", "-v"] if "--ptxas-v" in sys.argv else None
    print(build_library(force=force or bool(extra), verbose=True, extra_flags=extra))
