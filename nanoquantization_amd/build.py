"""Builds csrc/*.hip into nanoquantization_amd/libawq_hip.so for gfx950, csrc/hybrid/*.hip into libnq_hybrid.so, csrc/mx/*.hip into libnq_mx.so, and
csrc/torch_binding.cpp and csrc/mx/mx_binding.cpp (host code only: the PyTorch operator registration over the C ABIs) into
nanoquantization_amd/libawq_torch.so and libnq_mx_torch.so.

Usage: python -m nanoquantization_amd.build
"""
from __future__ import annotations

import glob
import os
import subprocess
import sys

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG_DIR, "csrc")
LIB_PATH = os.path.join(PKG_DIR, "libawq_hip.so")

HYBRID_CSRC = os.path.join(CSRC, "hybrid")
HYBRID_LIB_PATH = os.path.join(PKG_DIR, "libnq_hybrid.so")

MX_CSRC = os.path.join(CSRC, "mx")
MX_LIB_PATH = os.path.join(PKG_DIR, "libnq_mx.so")

TORCH_LIB_PATH = os.path.join(PKG_DIR, "libawq_torch.so")
MX_TORCH_LIB_PATH = os.path.join(PKG_DIR, "libnq_mx_torch.so")

ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")
HIPCC = os.environ.get("HIPCC", os.path.join(ROCM, "bin", "hipcc"))
CXX = os.environ.get("CXX", "g++")
FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    # packed-fp32 arithmetic is switched off for every kernel of this library
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
]


# per-source extra flags
EXTRA = {
    # keep MFMA results in VGPRs: the GEMV folds every accumulator into fp32 state right away,
    # AGPR destinations would cost a v_accvgpr_read per value and 4 more registers per wave
    "awq_gemv.hip": ["-mllvm", "-amdgpu-mfma-vgpr-form"],
    # the SLP vectoriser pairs the two k rows of the unpack into <2 x i32> and/or, which then no
    # longer select as one v_and_or_b32 each
    "awq_gemm_pipe.hip": ["-fno-slp-vectorize"],
    "awq_gemm_regb.hip": ["-fno-slp-vectorize"],
    "awq_gemm_rows.hip": ["-fno-slp-vectorize"],
}


def sources() -> list[str]:
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _run(cmd, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    proc = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    # the host pass does not know the device-only target feature and says so once per file
    out = "\n".join(l for l in proc.stdout.splitlines() if "packed-fp32-ops" not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{out}")
    if verbose and out.strip():
        print(out)


def _build_folder(csrc: str, name: str, lib: str, verbose: bool) -> str:
    """Compile csrc/*.hip (in parallel) and link them into `lib`."""
    from concurrent.futures import ThreadPoolExecutor

    objdir = os.path.join(PKG_DIR, "build", name)
    os.makedirs(objdir, exist_ok=True)
    compile_flags = [f for f in FLAGS if f != "-shared"]
    srcs = sorted(glob.glob(os.path.join(csrc, "*.hip")))
    objs = [os.path.join(objdir, os.path.basename(s) + ".o") for s in srcs]
    with ThreadPoolExecutor(max_workers=8) as pool:
        list(pool.map(lambda so: _run([HIPCC, *compile_flags, *EXTRA.get(os.path.basename(so[0]), []), "-c", so[0],
                                       "-o", so[1]], verbose), zip(srcs, objs)))
    part = f"{lib}.{os.getpid()}"       # a second process never sees half a library
    _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *objs, "-o", part], verbose)
    os.replace(part, lib)
    return lib


def build_hybrid(verbose: bool = True) -> str:
    """Compile csrc/hybrid/*.hip (in parallel) and link libnq_hybrid.so: all that the hybrid decoders need."""
    return _build_folder(HYBRID_CSRC, "hybrid", HYBRID_LIB_PATH, verbose)


def build_mx(verbose: bool = True) -> str:
    """libnq_mx.so from csrc/mx/*.hip, and its operators, libnq_mx_torch.so: all that the microscaled formats need."""
    _build_folder(MX_CSRC, "mx", MX_LIB_PATH, verbose)
    obj = os.path.join(PKG_DIR, "build", "mx", "mx_binding.o")
    _run(torch_binding_compile_cmd(obj, os.path.join(MX_CSRC, "mx_binding.cpp")), verbose)
    _run(torch_binding_link_cmd(obj, MX_TORCH_LIB_PATH, "nq_mx"), verbose)
    return MX_LIB_PATH


def ensure_hybrid() -> None:
    """Build libnq_hybrid.so if this checkout does not have it yet."""
    if not os.path.exists(HYBRID_LIB_PATH):
        build_hybrid(verbose=False)


def build(verbose: bool = True) -> str:
    """Compile every HIP source (in parallel) and link the shared libraries; returns the path of libawq_hip.so."""
    from concurrent.futures import ThreadPoolExecutor

    build_hybrid(verbose)
    build_mx(verbose)
    objdir = os.path.join(PKG_DIR, "build")
    os.makedirs(objdir, exist_ok=True)
    compile_flags = [f for f in FLAGS if f != "-shared"]
    jobs = []
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        jobs.append(([HIPCC, *compile_flags, *EXTRA.get(os.path.basename(src), []), "-c", src, "-o", obj], obj))
    with ThreadPoolExecutor(max_workers=min(4, len(jobs))) as pool:
        list(pool.map(lambda j: _run(j[0], verbose), jobs))
    with ThreadPoolExecutor(max_workers=2) as pool:
        # the operator binding has no device code: host compiler, torch headers; it only needs the C header
        binding = pool.submit(_run, torch_binding_compile_cmd(os.path.join(objdir, "torch_binding.o")), verbose)
        _run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", *[o for _, o in jobs], "-o", LIB_PATH], verbose)
        binding.result()
    _run(torch_binding_link_cmd(os.path.join(objdir, "torch_binding.o")), verbose)
    return LIB_PATH


def _torch_dirs():
    import torch
    root = os.path.dirname(torch.__file__)
    return ([os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include")],
            os.path.join(root, "lib"), int(torch._C._GLIBCXX_USE_CXX11_ABI))


def torch_binding_compile_cmd(obj: str, source: str = os.path.join(CSRC, "torch_binding.cpp")) -> list[str]:
    incs, _, abi = _torch_dirs()
    return [CXX, "-O2", "-fPIC", "-std=c++17", "-w", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *[f"-I{i}" for i in incs], f"-I{ROCM}/include",
            "-c", source, "-o", obj]


def torch_binding_link_cmd(obj: str, lib: str = TORCH_LIB_PATH, over: str = "awq_hip") -> list[str]:
    _, libdir, _ = _torch_dirs()
    return [CXX, "-shared", "-fPIC", obj, "-o", lib, f"-L{libdir}", "-ltorch", "-ltorch_cpu", "-lc10",
            "-lc10_hip", "-ltorch_hip", f"-L{PKG_DIR}", f"-l{over}", "-ldl", "-Wl,-rpath,$ORIGIN", f"-Wl,-rpath,{libdir}"]


if __name__ == "__main__":
    build()
    sys.exit(0)
