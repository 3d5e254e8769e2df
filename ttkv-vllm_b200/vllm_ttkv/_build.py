"""Build `libttkv_sm100.so` in-tree with nvcc for sm_100a (B200), and its torch binding
`_ttkv_torch.so` (csrc/ttkv_torch.cpp) with the host compiler."""
from __future__ import annotations

import os
import pathlib
import shutil
import subprocess

PKG = pathlib.Path(__file__).resolve().parents[1]          # the ttkv-vllm_b200 directory
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
OUT = PKG / "libttkv_sm100.so"
BINDING = PKG / "_ttkv_torch.so"
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def sources():
    return sorted(CSRC.glob("*.cu"))


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and pathlib.Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def up_to_date() -> bool:
    if not OUT.exists() or not BINDING.exists() or BINDING.stat().st_mtime < OUT.stat().st_mtime or \
            BINDING.stat().st_mtime < (CSRC / "ttkv_torch.cpp").stat().st_mtime:
        return False
    t = OUT.stat().st_mtime
    deps = sources() + sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    return all(p.stat().st_mtime <= t for p in deps)


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile every .cu under csrc/ into one shared library next to the package, and its binding."""
    if not force and up_to_date():
        return OUT
    cmd = [nvcc(), "--threads", "0", *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-shared",
           f"-I{INCLUDE}", f"-I{CSRC}", "-o", str(OUT) + ".tmp", *map(str, sources())]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    subprocess.run(cmd, check=True)
    os.replace(str(OUT) + ".tmp", OUT)
    build_binding()
    return OUT


def build_binding() -> pathlib.Path:
    """Compile the torch binding against the library that is there."""
    import sysconfig

    import torch
    home = pathlib.Path(torch.__file__).resolve().parent
    cuda = pathlib.Path(nvcc()).resolve().parents[1]
    inc = [home / "include", home / "include/torch/csrc/api/include", sysconfig.get_paths()["include"],
           cuda / "include", INCLUDE]
    subprocess.run(
        [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
         f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{d}" for d in inc),
         "-o", str(BINDING) + ".tmp", str(CSRC / "ttkv_torch.cpp"), f"-L{PKG}", f"-l:{OUT.name}",
         f"-L{home / 'lib'}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python",
         "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(str(BINDING) + ".tmp", BINDING)
    return BINDING


if __name__ == "__main__":
    print(build(force=True, verbose=True))
