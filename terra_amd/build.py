"""Builds ``terra_amd/libterra_swin.so`` from ``terra_amd/csrc`` with hipcc for gfx950,
and the host modules of the operators that have one beside it.

    python -m terra_amd.build

The library is written in-tree (it travels with the source tree to the GPU
host; nothing is JIT-compiled at run time).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SOURCES = ("abi.hip", "window_copy.hip", "window_attention.hip", "window_attention_bwd.hip", "swin_block.hip",
           "swin_mlp.hip", "linear.hip", "mlp_backward.hip", "weight_grad.hip", "linear_short.hip", "block_f32.hip",
           "dropout.hip", "residual_norm.hip", "residual_norm_f32_f32.hip", "residual_norm_bf16_bf16.hip",
           "residual_norm_bf16_f32.hip", "residual_norm_f16_f16.hip", "residual_norm_f16_f32.hip", "layer_norm.hip", "layer_norm_f32_f32.hip",
           "layer_norm_f32_bf16.hip", "layer_norm_f32_f16.hip", "layer_norm_bf16_bf16.hip", "layer_norm_bf16_f32.hip",
           "layer_norm_f16_f16.hip", "layer_norm_f16_f32.hip", "rotary.hip", "optimizer.hip")
ARCH = "gfx950"

HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # Packed-fp32 VALU ops are kept out of the device code.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # MFMA results in arch VGPRs (no AGPR round trip): keeps the attention
    # kernel at <= 128 VGPRs, i.e. 4 waves per SIMD.
    "-mllvm", "-amdgpu-mfma-vgpr-form=1",
    "-Wall",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (ROCm toolchain required to build libterra_swin.so)")


def _run(cmd, verbose: bool) -> str:
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    out = "\n".join(line for line in proc.stdout.splitlines() if "packed-fp32-ops" not in line)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{out}")
    return out


# Host-side AddressSanitizer (the C-ABI validation code; device code is built
# as usual): each flag applies to the host compilation only.
ASAN_HOST_FLAGS = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fno-omit-frame-pointer"]
ASAN_LIB_PATH = os.path.join(HERE, "libterra_swin_asan.so")


def build_library(verbose: bool = False, jobs: int = 0, asan_host: bool = False) -> str:
    """Compile every HIP source (one hipcc process per source, in parallel)
    and link them into the shared library; returns its path.  ``asan_host``
    builds ``libterra_swin_asan.so`` instead, its host code under
    AddressSanitizer (load it with the sanitizer runtime preloaded and
    TERRA_SWIN_LIB naming it)."""
    from concurrent.futures import ThreadPoolExecutor

    from ._lib import LIB_PATH as default_path  # noqa: WPS433 (path only; does not open the library)

    LIB_PATH = ASAN_LIB_PATH if asan_host else default_path
    extra = ASAN_HOST_FLAGS if asan_host else []
    jobs = jobs or min(len(SOURCES), os.cpu_count() or 1, 8)
    compile_flags = [f for f in HIPCC_FLAGS if f != "-shared"] + extra
    with tempfile.TemporaryDirectory(prefix="_build.", dir=HERE) as tmpdir:
        objs = [os.path.join(tmpdir, os.path.splitext(s)[0] + ".o") for s in SOURCES]
        cmds = [[hipcc(), *compile_flags, "-c", os.path.join(CSRC, s), "-o", o] for s, o in zip(SOURCES, objs)]
        with ThreadPoolExecutor(max_workers=jobs) as pool:
            outs = list(pool.map(lambda c: _run(c, verbose), cmds))
        fd, tmp = tempfile.mkstemp(prefix="libterra_swin.", suffix=".so.tmp", dir=HERE)
        os.close(fd)
        try:
            outs.append(_run([hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", *extra, *objs, "-o", tmp],
                             verbose))
        except RuntimeError:
            os.unlink(tmp)
            raise
    if verbose:
        for out in outs:
            if out.strip():
                print(out, flush=True)
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


# The host modules: name -> source, against torch's headers.
BINDINGS = {"_regularize": "regularize_binding.cpp", "_training": "training_binding.cpp"}


def build_binding(verbose: bool = False, name: str = "_regularize") -> str:
    """Compile a host module (of the regularised operators, or ``_training`` of
    the norms, rotary positions and the optimizer's step) into ``terra_amd/<name>.so``; returns its path."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension

    path = os.path.join(HERE, f"{name}.so")
    root = os.path.dirname(torch.__file__)
    cmd = [hipcc(), "-x", "c++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
           *(f"-isystem{d}" for d in [*cpp_extension.include_paths(), "/opt/rocm/include",
                                      sysconfig.get_paths()["include"]]),
           os.path.join(CSRC, BINDINGS[name]), f"-L{os.path.join(root, 'lib')}", "-ltorch_python",
           "-ltorch_cpu", "-ltorch", "-lc10", "-lc10_hip"]
    fd, tmp = tempfile.mkstemp(prefix=f"{name}.", suffix=".so.tmp", dir=HERE)
    os.close(fd)
    try:
        _run([*cmd, "-o", tmp], verbose)
    except RuntimeError:
        os.unlink(tmp)
        raise
    os.chmod(tmp, 0o755)
    os.replace(tmp, path)
    return path


def build_bindings(verbose: bool = False) -> list:
    """Compile every host module, side by side; returns their paths."""
    from concurrent.futures import ThreadPoolExecutor

    with ThreadPoolExecutor() as pool:
        return list(pool.map(lambda name: build_binding(verbose, name), BINDINGS))


def asan_runtime() -> str:
    """Path of the clang AddressSanitizer runtime that hipcc links against."""
    out = subprocess.run([hipcc(), "-print-file-name=libclang_rt.asan-x86_64.so"], stdout=subprocess.PIPE,
                         stderr=subprocess.DEVNULL, text=True).stdout.strip()
    if out and os.path.isabs(out) and os.path.exists(out):
        return out
    import glob

    for cand in sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so")):
        return cand
    raise RuntimeError("clang AddressSanitizer runtime not found")


if __name__ == "__main__":
    path = build_library(verbose=True, asan_host="--asan-host" in sys.argv)
    print(path)
    if "--asan-host" not in sys.argv:
        for path in build_bindings(verbose=True):
            print(path)
    sys.exit(0)
