"""Build recipe for libmt_flce.so (gfx950 only).

The library is five translation units (csrc/flce_capi.hip: the loss;
csrc/attn_capi.hip: attention; csrc/step_capi.hip: residual norms and clipping;
csrc/layer_capi.hip: token embedding and layer norm; csrc/update_capi.hip:
orthogonalised updates; each includes its kernels' headers) compiled side by side with hipcc for gfx950 and linked into the package
directory, so it travels with the source tree.  `python -m mini_trainer_amd.build` rebuilds it.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libmt_flce.so"
SOURCES = [CSRC / "flce_capi.hip", CSRC / "attn_capi.hip", CSRC / "step_capi.hip",
           CSRC / "layer_capi.hip", CSRC / "update_capi.hip"]
DEPENDS = sorted(CSRC.glob("*.h")) + SOURCES + [PKG_DIR.parent / "include" / "mt_flce.h"]

# The autograd nodes in C++ (csrc/torch_ops.cpp): a Python module built against this
# torch, which is handed the library's functions when both are loaded.
TORCH_SOURCE = CSRC / "torch_ops.cpp"
TORCH_PATH = PKG_DIR / "_mt_torch.so"
TORCH_DEPENDS = [TORCH_SOURCE, PKG_DIR.parent / "include" / "mt_flce.h"]

ARCH = "gfx950"
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    # Packed fp32 VALU ops stay disabled in all device code of this library.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required to build libmt_flce.so)")


SAN_LIB_PATH = PKG_DIR / "_build" / "libmt_flce_san.so"
# The CPU tests' build: AddressSanitizer and UndefinedBehaviorSanitizer on
# the host pass only (the device code is compiled plainly, at -O1, and never
# runs: the CPU tests exercise the argument checks, planners and error
# paths, on a machine without a GPU).
SAN_FLAGS = [
    f"--offload-arch={ARCH}", "-O1", "-g", "-std=c++17", "-fPIC",
    "-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
    "-Xarch_host", "-fno-sanitize-recover=all", "-Xarch_host", "-fno-omit-frame-pointer",
    "-Xarch_device", "-g0",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


def _older(built: Path, sources: list) -> bool:
    """Whether a build is missing, or older than one of its sources."""
    if not built.exists():
        return True
    t = built.stat().st_mtime
    return any(p.stat().st_mtime > t for p in sources if p.exists())


def san_is_stale() -> bool:
    return _older(SAN_LIB_PATH, DEPENDS)


def _compile(out: Path, flags: list, verbose: bool) -> str:
    """Compile every source with `flags` at the same time, link them into `out`
    and return what the compiler said."""
    objects = PKG_DIR / "_build"
    objects.mkdir(exist_ok=True)
    steps = []
    for src in SOURCES:
        obj = objects / f"{out.stem}-{src.stem}.o"
        cmd = [hipcc(), *flags, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        steps.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                            text=True)))
    said = [p.communicate()[0] for _, p in steps]  # all have ended before one may raise
    for (_, p), text in zip(steps, said):
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed ({p.returncode}):\n{text}")
    tmp = out.with_suffix(".so.tmp")
    link = [hipcc(), *flags, "-shared", "-o", str(tmp), *(str(obj) for obj, _ in steps)]
    proc = subprocess.run(link, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc (link) failed ({proc.returncode}):\n{proc.stderr}")
    os.replace(tmp, out)
    return "".join(said)


def build_sanitized(verbose: bool = False) -> Path:
    """Compile the sanitized test build (_build/libmt_flce_san.so).  Always
    recompiles (about a minute).  Load it with the clang ASan runtime
    preloaded."""
    _compile(SAN_LIB_PATH, SAN_FLAGS, verbose)
    return SAN_LIB_PATH


def asan_runtime() -> Path:
    """The clang ASan runtime matching hipcc (to LD_PRELOAD into Python)."""
    clang = Path(hipcc()).resolve().parent.parent / "llvm" / "bin" / "clang"
    if not clang.exists():
        clang = Path("/opt/rocm/llvm/bin/clang")
    out = subprocess.run([str(clang), "-print-file-name=libclang_rt.asan-x86_64.so"],
                         capture_output=True, text=True).stdout.strip()
    return Path(out)


def build_library(verbose: bool = False) -> Path:
    """Compile libmt_flce.so for gfx950.  Always recompiles."""
    said = _compile(LIB_PATH, HIPCC_FLAGS, verbose)
    # hipcc's host pass does not know the packed-fp32 feature; drop that noise.
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in said.splitlines() if noise not in l)
    if verbose and err.strip():
        print(err, file=sys.stderr)
    return LIB_PATH


def build_torch_ops(verbose: bool = False) -> Path:
    """Compile _mt_torch.so with the host compiler.  Always recompiles."""
    import sysconfig

    import torch

    root = Path(torch.__file__).resolve().parent
    include = [root / "include", root / "include" / "torch" / "csrc" / "api" / "include",
               sysconfig.get_paths()["include"]]
    tmp = TORCH_PATH.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", *(f"-I{i}" for i in include),
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-fvisibility=hidden",
           f'-DMT_TORCH_VERSION="{torch.__version__}"',
           str(TORCH_SOURCE), "-o", str(tmp), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch",
           "-ltorch_cpu", "-lc10"]
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed ({proc.returncode}):\n{proc.stderr}")
    os.replace(tmp, TORCH_PATH)
    return TORCH_PATH


def is_stale() -> bool:
    """Of the library and the autograd nodes."""
    return _older(LIB_PATH, DEPENDS) or _older(TORCH_PATH, TORCH_DEPENDS)


if __name__ == "__main__":
    print(build_library(verbose=True))
    print(build_torch_ops(verbose=True))
