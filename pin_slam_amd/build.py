"""Build the gfx950 shared library in-tree, pin_slam_amd/libpin_slam_amd.so, and beside it
libpin_slam_torch.so (csrc/pin_torch.cpp, host code against torch's headers).

hipcc cross-compiles for gfx950 without a GPU, so this runs in the build
container; the resulting .so travels to the GPU box with the repo snapshot.
"""
import glob
import os
import shutil
import subprocess
import sys
import sysconfig
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
LIB = os.path.join(HERE, "libpin_slam_amd.so")
TORCH_LIB = os.path.join(HERE, "libpin_slam_torch.so")
TORCH_SOURCE = os.path.join(HERE, "csrc", "pin_torch.cpp")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    # every elementwise op rounds like the reference's unfused ATen ops; FMAs are explicit
    "-ffp-contract=off",
    # no packed-f32 instructions (v_pk_fma_f32 and its like): some of their forms have given wrong
    # values now and then on this hardware.  The host pass warns that it does not know the feature.
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]


def sources():
    return sorted(glob.glob(os.path.join(HERE, "csrc", "*.hip")))


def _stale():
    if not os.path.exists(LIB) or not os.path.exists(TORCH_LIB):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(TORCH_LIB))
    deps = sources() + glob.glob(os.path.join(HERE, "csrc", "*.h")) + [TORCH_SOURCE, os.path.join(ROOT, "include", "pin_slam_amd.h")]
    return any(os.path.getmtime(d) > t for d in deps)


def _torch_command(out):
    import torch
    from torch.utils import cpp_extension
    libs = os.path.join(os.path.dirname(torch.__file__), "lib")
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM",
            "-isystem/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
            *[f"-isystem{p}" for p in cpp_extension.include_paths()], f"-isystem{sysconfig.get_paths()['include']}",
            TORCH_SOURCE, f"-L{libs}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_hip", "-o", out]


def build(force: bool = False, verbose: bool = False, extra=(), out: str = None) -> str:
    """Compile every csrc/*.hip into one shared library (``out`` defaults to the in-tree LIB;
    ``extra`` adds compiler flags, e.g. -D switches for experiment variants)."""
    out = out or LIB
    if out == LIB and not force and not _stale():
        return LIB
    # one object per source, compiled in parallel (objects outside the tree), then one link
    objdir = tempfile.mkdtemp(prefix="pin_slam_amd_obj_")
    inc = ["-I", os.path.join(ROOT, "include"), "-I", os.path.join(HERE, "csrc")]
    try:
        procs = []
        objs = []
        if out == LIB:
            cmd = _torch_command(TORCH_LIB + ".tmp")
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            procs.append((cmd, subprocess.Popen(cmd)))
        for src in sources():
            obj = os.path.join(objdir, os.path.basename(src) + ".o")
            cmd = [HIPCC, *[f for f in FLAGS if f != "-shared"], *extra, *inc, "-c", src, "-o", obj]
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            procs.append((cmd, subprocess.Popen(cmd)))
            objs.append(obj)
        for cmd, p in procs:
            if p.wait() != 0:
                raise subprocess.CalledProcessError(p.returncode, cmd)
        subprocess.run([HIPCC, *FLAGS, *objs, "-o", out + ".tmp"], check=True)
    finally:
        shutil.rmtree(objdir, ignore_errors=True)
    os.replace(out + ".tmp", out)
    if out == LIB:
        os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    return out


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
