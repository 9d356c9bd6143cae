"""Build the gfx950 KDA library in-tree: ``axiom_amd/libkda_mi355x.so``.

Every HIP source under ``axiom_amd/csrc`` is compiled with hipcc for gfx950
only, then linked into one shared library whose exported functions are the C
ABI of ``include/kda_mi355x.h`` and ``include/latent_mi355x.h`` and the package's
own entry points (``_lib._PRIVATE``, declared in ``csrc/kda_internal.h``); the
torch binding of the latent attention, ``_latent_torch.so``, is host C++ over
that library.  Run ``python -m axiom_amd.build`` or call :func:`build`.
"""

from __future__ import annotations

import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libkda_mi355x.so"
BINDING = PKG / "_latent_torch.so"
INCLUDE = PKG.parent / "include"

ARCH = "gfx950"
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fvisibility=hidden",
    # packed fp32 VALU ops are kept out of every kernel of this library
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]
SOURCES = ["kda_chunk.hip", "kda_varlen.hip", "kda_decode.hip", "kda_bwd.hip", "kda_ut.hip", "kda_prologue.hip",
           "kda_latent_fwd.hip", "kda_latent_bwd.hip", "kda_latent_decode.hip", "kda_latent_api.hip", "kda_api.hip"]


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found: the KDA library needs ROCm's hipcc to build")


def _compile(src: Path, obj: Path, hipcc: str) -> None:
    cmd = [hipcc, *HIPCC_FLAGS, f"-I{INCLUDE}", f"-I{CSRC}", "-c", str(src), "-o", str(obj)]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{p.stderr}")


def _compile_binding(obj: Path, hipcc: str) -> None:
    """Host C++ against torch's headers (no kernel in it)."""
    import torch
    from torch.utils.cpp_extension import include_paths
    inc = [f"-I{p}" for p in (*include_paths(), sysconfig.get_paths()["include"], INCLUDE, Path(hipcc).resolve().parents[1] / "include")]
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           "-DTORCH_EXTENSION_NAME=_latent_torch", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", *inc,
           "-c", str(CSRC / "latent_torch.cpp"), "-o", str(obj)]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"g++ failed for latent_torch.cpp:\n{p.stderr}")


def _link_binding(obj: Path) -> None:
    import torch
    libs = Path(torch.__file__).parent / "lib"
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [shutil.which("g++") or "g++", "-shared", "-o", str(tmp), str(obj), f"-L{PKG}", "-lkda_mi355x", f"-L{libs}", "-lc10",
           "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN"]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"link of {BINDING.name} failed:\n{p.stderr}")
    os.replace(tmp, BINDING)


def build(verbose: bool = False) -> Path:
    """Compile all sources, link ``libkda_mi355x.so``, then its torch binding; returns the library's path.

    The library needs nothing of torch: it is in place before the binding is
    linked, and where torch is not importable the binding is left out.
    """
    hipcc = _hipcc()
    BUILD.mkdir(exist_ok=True)
    binding_obj = BUILD / "latent_torch.o"
    objs = [BUILD / (s.replace(".hip", ".o")) for s in SOURCES]
    with_torch = importlib.util.find_spec("torch") is not None
    with ThreadPoolExecutor(max_workers=min(len(SOURCES) + 1, os.cpu_count() or 1)) as ex:
        binding = ex.submit(_compile_binding, binding_obj, hipcc) if with_torch else None
        list(ex.map(lambda so: _compile(CSRC / so[0], so[1], hipcc), zip(SOURCES, objs)))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"link failed:\n{p.stderr}")
    os.replace(tmp, LIB)
    if binding is None:
        print(f"torch is not importable: {BINDING.name} (the torch binding of the latent attention) is not built", file=sys.stderr)
    else:
        binding.result()
        _link_binding(binding_obj)
    if verbose:
        print(f"built {LIB}")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)
