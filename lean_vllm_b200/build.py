"""Builds libkvx.so in-tree for sm_100a (B200) with nvcc, and the module that calls it from torch tensors:
`python -m lean_vllm_b200.build`."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
SOURCES = [os.path.join(CSRC, name) for name in ("kvx.cu", "rotary.cu", "attention.cu", "attention_tiles.cu")]
HEADERS = [os.path.join(ROOT, "include", "kvx.h"),
           *(os.path.join(CSRC, name) for name in sorted(os.listdir(CSRC)) if name.endswith(".cuh"))]
OUTPUT = os.path.join(HERE, "libkvx.so")
CALLS_SOURCE = os.path.join(CSRC, "calls.cpp")
CALLS = os.path.join(HERE, "_calls" + sysconfig.get_config_var("EXT_SUFFIX"))
CALLS_TORCH = CALLS + ".torch"  # the torch version it was built against

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-warn-spills",
]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(path):
        raise RuntimeError("nvcc not found; the CUDA toolkit is needed to build libkvx.so")
    return path


def stale(output: str = OUTPUT, sources: list[str] | None = None) -> bool:
    if not os.path.exists(output):
        return True
    built = os.path.getmtime(output)
    return any(os.path.getmtime(f) > built for f in (sources or SOURCES + HEADERS))


def build_calls(force: bool = False) -> str:
    """The binding of the calls a decode step makes per layer (csrc/calls.cpp), with g++ against torch's headers."""
    import torch
    from torch.utils import cpp_extension

    if not force and not stale(CALLS, [CALLS_SOURCE, HEADERS[0]]) and os.path.exists(CALLS_TORCH):
        with open(CALLS_TORCH) as f:
            if f.read() == torch.__version__:
                return CALLS
    cuda = os.path.dirname(os.path.dirname(nvcc()))
    includes = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], os.path.join(cuda, "include"),
                os.path.join(ROOT, "include")]
    libraries = cpp_extension.library_paths()
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           f'-DKVX_TORCH_VERSION="{torch.__version__}"', *(f"-I{i}" for i in includes), "-o", CALLS + ".tmp", CALLS_SOURCE, *(f"-L{d}" for d in libraries),
           "-lc10", "-ltorch_cpu", "-lc10_cuda", "-ltorch_python"]
    subprocess.run(cmd, check=True)
    os.replace(CALLS + ".tmp", CALLS)
    with open(CALLS_TORCH, "w") as f:
        f.write(torch.__version__)
    return CALLS


def build(force: bool = False, verbose: bool = False) -> str:
    build_calls(force)
    if not force and not stale():
        return OUTPUT
    # One object per source, compiled side by side, then linked; objects are rebuilt together with the library.
    with tempfile.TemporaryDirectory(prefix="kvx_build_") as work:
        objects = [os.path.join(work, os.path.basename(source) + ".o") for source in SOURCES]
        compiles = [[nvcc(), *(["-Xptxas=-v"] if verbose else []), *NVCC_FLAGS, "-I", os.path.join(ROOT, "include"),
                     "-c", "-o", obj, source] for source, obj in zip(SOURCES, objects)]
        if verbose:
            print("\n".join(" ".join(cmd) for cmd in compiles))
        running = [subprocess.Popen(cmd) for cmd in compiles]
        codes = [p.wait() for p in running]
        for code, cmd in zip(codes, compiles):
            if code:
                raise subprocess.CalledProcessError(code, cmd)
        subprocess.run([nvcc(), *NVCC_FLAGS, "-shared", "-o", OUTPUT + ".tmp", *objects], check=True)
    os.replace(OUTPUT + ".tmp", OUTPUT)
    return OUTPUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
