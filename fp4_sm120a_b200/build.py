"""Build the in-tree CUDA library libnvfp4_b200.so for sm_100a with nvcc, and the
tensor-level binding _torch_binding.*.so against torch's headers with the host
compiler.

Both are built next to this file so that they travel with the source
tree; nothing is installed into site-packages.  The library needs nvcc alone
(`python fp4_sm120a_b200/build.py` imports no package): where the binding cannot be
built, for want of torch, its headers or g++, the library is there all the same.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import Optional

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
LIB = PKG / "libnvfp4_b200.so"
OBJDIR = PKG / "_build"
BINDING_SOURCE = CSRC / "torch_binding.cpp"

# The system's compiler, whatever CXX says: the binding must share torch's
# libstdc++ (exceptions and streams cross between the two), and another compiler may
# link a copy of its own.
CXX = "g++"
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
SOURCES = ["rht_gemm_sm100.cu", "sr_kernels.cu", "fp8_kernels.cu", "fp8_kernels_loose.cu",
           "gemm_nvfp4_sm100.cu", "gemm_nvfp4_wide_sm100.cu", "layernorm.cu", "adamw.cu"]
FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC,-fvisibility=hidden",
    "-Xptxas", "-v",
    f"-I{INCLUDE}", f"-I{CSRC}",
]


def _deps() -> list[Path]:
    return sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + \
        sorted(INCLUDE.glob("*.h")) + sorted(INCLUDE.glob("*.cuh"))


def _stale(target: Path, deps: list[Path]) -> bool:
    return not target.exists() or any(d.stat().st_mtime > target.stat().st_mtime for d in deps)


def _binding_deps() -> list[Path]:
    return [BINDING_SOURCE, INCLUDE / "nvfp4_b200.h"]


def binding_path() -> Optional[Path]:
    """The binding's file, named by the Python and the torch it is built against and
    for (under others it is another file); None without torch."""
    try:
        import torch
    except ImportError:
        return None
    return PKG / f"_torch_binding.{sysconfig.get_config_var('SOABI')}-torch{torch.__version__}.so"


def needs_build() -> bool:
    binding = binding_path()
    return _stale(LIB, _deps()) or (binding is not None and _stale(binding, _binding_deps()))


def _run(cmd: list[str], what: str, verbose: bool = False) -> None:
    r = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or r.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
    if r.returncode != 0:
        raise RuntimeError(f"{what} failed")


def _build_binding(binding: Path, verbose: bool) -> None:
    """Needs LIB: the binding links against it (found beside it at run time)."""
    import torch
    root = Path(torch.__file__).resolve().parent
    tmp = binding.with_suffix(".so.tmp")
    _run([CXX, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
          f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
          f"-I{root / 'include'}", f"-I{root / 'include/torch/csrc/api/include'}",
          f"-I{Path(NVCC).resolve().parent.parent / 'include'}",
          f"-I{sysconfig.get_paths()['include']}", f"-I{INCLUDE}", str(BINDING_SOURCE),
          "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch_cuda", "-ltorch_cpu",
          "-ltorch", "-lc10_cuda", "-lc10", f"-L{PKG}", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"],
         "building the torch binding", verbose)
    os.replace(tmp, binding)


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not needs_build():
        return LIB
    OBJDIR.mkdir(exist_ok=True)

    headers = [d for d in _deps() if d.suffix != ".cu"]

    def compile_one(src: str) -> str:
        obj = OBJDIR / (Path(src).stem + ".o")
        if not force and not _stale(obj, [CSRC / src, *headers]):
            return str(obj)
        _run([NVCC, *FLAGS, "-c", str(CSRC / src), "-o", str(obj)], f"nvcc on {src}", verbose)
        return str(obj)

    if force or _stale(LIB, _deps()):
        with ThreadPoolExecutor(max_workers=len(SOURCES)) as pool:
            objs = list(pool.map(compile_one, SOURCES))
        tmp = LIB.with_suffix(".so.tmp")
        _run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", *objs, "-o",
              str(tmp)], "link")
        os.replace(tmp, LIB)
    binding = binding_path()
    if binding is None:
        sys.stderr.write("no torch: the tensor-level binding is not built\n")
    elif force or _stale(binding, _binding_deps()):
        # An old file would be imported as it is; the tensor-level calls raise without one.
        binding.unlink(missing_ok=True)
        try:
            _build_binding(binding, verbose)
        except (RuntimeError, OSError) as e:
            sys.stderr.write(f"the tensor-level binding is not built: {e}\n")
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
