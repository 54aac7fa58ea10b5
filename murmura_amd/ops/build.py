"""Build the HIP extension IN-TREE for gfx950.

``python -m murmura_amd.ops.build`` compiles the sources of hip/ with hipcc
(one process a file, side by side) and links ``_murmura_hip.so`` next to this
file, so that it goes wherever the tree goes (never a JIT cache under
~/.cache). hipcc cross-compiles without a GPU, so this runs on a machine of
CPUs too. The sources are HIP as they stand: they are handed to
the compiler directly, with torch's include paths and defines.
"""

from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).parent
SOURCES = [
    PKG_DIR / "hip" / name
    for name in ("murmura_kernels.hip", "group_norm.hip", "adamw.hip", "linear_act.hip")
]
BUILD_DIR = PKG_DIR / "_build"
OUT_SO = PKG_DIR / "_murmura_hip.so"


def _flags() -> list:
    import torch
    from torch.utils import cpp_extension

    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    includes = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    return [
        "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "--offload-arch=gfx950",
        # packed fp32 instructions are left out: some of their forms have given
        # wrong results on this hardware
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DHIPBLAS_V2", "-DCUDA_HAS_FP16=1",
        "-DTORCH_API_INCLUDE_EXTENSION_H", "-DTORCH_EXTENSION_NAME=_murmura_hip",
        f"-D_GLIBCXX_USE_CXX11_ABI={abi}", "-Wno-unused-command-line-argument",
        *[f"-isystem{p}" for p in includes],
    ]


def _run(cmd: list, verbose: bool) -> None:
    if verbose:
        print(" ".join(cmd), flush=True)
    done = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if verbose and done.stdout:
        print(done.stdout, flush=True)
    if done.returncode:
        raise RuntimeError(f"{cmd[0]} failed ({done.returncode}):\n{done.stdout[-8000:]}")


def build(verbose: bool = False) -> Path:
    from torch.utils import cpp_extension

    hipcc = str(Path(cpp_extension.ROCM_HOME or "/opt/rocm") / "bin" / "hipcc")
    BUILD_DIR.mkdir(exist_ok=True)
    flags = _flags()
    objects = [BUILD_DIR / (src.stem + ".o") for src in SOURCES]
    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        list(pool.map(
            lambda so: _run([hipcc, *flags, "-c", str(so[0]), "-o", str(so[1])], verbose),
            zip(SOURCES, objects),
        ))
    built = BUILD_DIR / "_murmura_hip.so"
    libs = [f"-L{p}" for p in cpp_extension.library_paths("cuda")]
    _run([hipcc, "-shared", "-fPIC", "--offload-arch=gfx950", *map(str, objects), *libs,
          "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch", "-ltorch_python",
          "-o", str(built)], verbose)
    # in place at once: a reader sees the old library or the new one
    staged = OUT_SO.with_name("_murmura_hip.new")
    staged.write_bytes(built.read_bytes())
    staged.chmod(0o755)
    os.replace(staged, OUT_SO)
    return OUT_SO


if __name__ == "__main__":
    so = build(verbose="-v" in sys.argv)
    print(f"built {so}")
