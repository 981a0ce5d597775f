"""Build libcc1d_b200.so (the C-ABI library of the causal_conv1d B200 kernels) and _block.so
(the PyTorch binding of its recurrent-block operators).

    python cute-causal-conv1d_b200/cc1d_build.py [--force] [--verbose]

Compiles every kernel file for sm_100a only (``-gencode arch=compute_100a,code=sm_100a``)
with nvcc, in parallel; the per-element-type kernel files are compiled once per type.
The library is written next to the Python package (``causal_conv1d/libcc1d_b200.so``),
in the source tree, and is rebuilt only when a source or header is newer.  So is the
binding, which g++ compiles against the headers of the installed PyTorch; the library itself
needs no PyTorch, and is built alone where there is none.
"""

from __future__ import annotations

import argparse
import importlib.util
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")
BUILD = os.path.join(HERE, "_build")
LIB = os.path.join(HERE, "causal_conv1d", "libcc1d_b200.so")
# the PyTorch binding of the recurrent-block operators, an extension module on top of LIB
BINDING = os.path.join(HERE, "causal_conv1d", "_block.so")

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + [
    "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC,-O2",
    "-I" + INCLUDE, "-I" + CSRC,
]

# (source, extra defines, object name)
UNITS = [
    ("cc1d_abi.cu", [], "cc1d_abi.o"),
    ("cc1d_update.cu", [], "cc1d_update.o"),
    ("cc1d_decode.cu", [], "cc1d_decode.o"),
    ("cc1d_static.cu", [], "cc1d_static.o"),
    ("cc1d_block_abi.cu", [], "cc1d_block_abi.o"),
    ("cc1d_selective_abi.cu", [], "cc1d_selective_abi.o"),
    ("cc1d_beam.cu", [], "cc1d_beam.o"),
    ("cc1d_beam_abi.cu", [], "cc1d_beam_abi.o"),
] + [
    (src, [f"-DCC1D_DT={dt}"], f"{src[:-3]}_{name}.o")
    for src in ("cc1d_fwd.cu", "cc1d_bwd.cu", "cc1d_rows.cu", "cc1d_rowwalk.cu",
                "cc1d_recurrence.cu", "cc1d_recurrence_update.cu", "cc1d_add_norm.cu",
                "cc1d_selective_fwd.cu", "cc1d_selective_bwd.cu", "cc1d_selective_update.cu")
    for dt, name in ((0, "f32"), (1, "f16"), (2, "bf16"))
]


def nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(exe):
        raise RuntimeError("nvcc not found; the CUDA toolkit is required to build libcc1d_b200.so")
    return exe


def _inputs():
    files = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    files += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    files.append(os.path.abspath(__file__))
    return files


def has_torch() -> bool:
    return importlib.util.find_spec("torch") is not None


def up_to_date() -> bool:
    built = [LIB, BINDING] if has_torch() else [LIB]
    if not all(os.path.exists(f) for f in built):
        return False
    oldest = min(os.path.getmtime(f) for f in built)
    return all(os.path.getmtime(f) <= oldest for f in _inputs())


def compile_binding(obj: str) -> None:
    """cc1d_block_torch.cpp -> obj, with the installed PyTorch's headers and C++ ABI."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    cuda = os.path.dirname(os.path.dirname(nvcc()))
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-c", os.path.join(CSRC, "cc1d_block_torch.cpp"), "-o", obj,
           "-DTORCH_EXTENSION_NAME=_block", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I" + INCLUDE, "-I" + os.path.join(cuda, "include"), "-I" + sysconfig.get_path("include")]
    cmd += ["-isystem" + d for d in cpp_extension.include_paths()]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"g++ failed for cc1d_block_torch.cpp:\n{res.stdout}\n{res.stderr}")


def link_binding(obj: str) -> None:
    from torch.utils import cpp_extension

    tmp = BINDING + ".tmp"
    cmd = ["g++", "-shared", "-o", tmp, obj, "-Wl,-rpath,$ORIGIN"]
    cmd += ["-L" + d for d in (os.path.dirname(LIB), *cpp_extension.library_paths())]
    cmd += ["-l:" + os.path.basename(LIB), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link of _block.so failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, BINDING)


def build(force: bool = False, verbose: bool = False) -> str:
    if not force and up_to_date():
        return LIB
    os.makedirs(BUILD, exist_ok=True)
    exe = nvcc()

    def compile_unit(unit):
        src, defs, obj = unit
        cmd = [exe] + NVCC_FLAGS + defs + ["-c", os.path.join(CSRC, src), "-o", os.path.join(BUILD, obj)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError(f"nvcc failed for {src} {defs}:\n{res.stdout}\n{res.stderr}")
        return res.stderr

    workers = max(1, min(len(UNITS), os.cpu_count() or 4))
    binding_obj = os.path.join(BUILD, "cc1d_block_torch.o")
    with ThreadPoolExecutor(workers) as pool:
        binding = pool.submit(compile_binding, binding_obj) if has_torch() else None
        logs = list(pool.map(compile_unit, UNITS))
    if verbose:
        for log in logs:
            sys.stderr.write(log)
    objs = [os.path.join(BUILD, u[2]) for u in UNITS]
    tmp = LIB + ".tmp"
    cmd = [exe] + ARCH + ["-shared", "-o", tmp] + objs
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stdout}\n{res.stderr}")
    os.replace(tmp, LIB)
    if binding is None:
        sys.stderr.write("cc1d_build: no PyTorch here, so its binding _block.so is not built\n")
    else:
        binding.result()
        link_binding(binding_obj)
    return LIB


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    args = ap.parse_args()
    print(build(force=args.force, verbose=args.verbose))


if __name__ == "__main__":
    main()
