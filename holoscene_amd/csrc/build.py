"""Build libholoscene_hip.so for gfx950 in-tree (hipcc cross-compiles without a GPU), and _row_autograd.so, the autograd nodes of the row operators
(host code against PyTorch's C++ interface).

    python -m holoscene_amd.csrc.build [--force]

The shared library lands next to the sources (git-ignored, but it travels to the GPU
box with the gpurun snapshot).  There is exactly one target: MI355X / gfx950.
"""
import glob
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
LIB = os.path.join(HERE, "libholoscene_hip.so")
NODES = os.path.join(HERE, "_row_autograd.so")
ARCH = "gfx950"
# -ffp-contract=off: the encoder must round exactly like the CPU oracle (no fused multiply-adds).
# -packed-fp32-ops: no packed fp32 instructions (v_pk_add / mul / fma_f32), some forms of which have given wrong results on this hardware;
#   the default training iteration is 0.3 % slower without them (1.530 against 1.526 ms median, alternating runs).  The host pass
#   does not know the feature and says so: harmless.
FLAGS = ["-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-munsafe-fp-atomics", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def sources():
    return sorted(glob.glob(os.path.join(HERE, "*.hip")))


def _nodes_command():
    import torch
    base = os.path.dirname(torch.__file__)
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"), "/opt/rocm/include", sysconfig.get_paths()["include"]]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-DUSE_ROCM=1", "-D__HIP_PLATFORM_AMD__=1", "-DTORCH_API_INCLUDE_EXTENSION_H",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", "-I", os.path.join(ROOT, "include"), *[f for p in include for f in ("-isystem", p)],
            os.path.join(HERE, "row_autograd.cpp"), "-o", NODES, "-L", os.path.join(base, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch", "-ltorch_python"]


def _stale():
    if not os.path.exists(LIB) or not os.path.exists(NODES):
        return True
    t = min(os.path.getmtime(LIB), os.path.getmtime(NODES))
    deps = sources() + [os.path.join(HERE, "row_autograd.cpp")] + glob.glob(os.path.join(HERE, "*.h")) + glob.glob(os.path.join(ROOT, "include", "*.h")) + [__file__]
    return any(os.path.getmtime(p) > t for p in deps)


def build(force=False, verbose=False, variant=None, extra_flags=()):
    """variant: build a SECOND library `libholoscene_hip_<variant>.so` with extra compile flags (kernel A/B runs on one box:
    HOLOSCENE_LIB=<that path> selects it in hashencoder/backend.py); its objects live in their own directory."""
    if variant is None and not force and not _stale():
        return LIB
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = []
    procs = []
    lib = LIB if variant is None else os.path.join(HERE, f"libholoscene_hip_{variant}.so")
    objdir = HERE if variant is None else os.path.join(HERE, f"obj_{variant}")
    os.makedirs(objdir, exist_ok=True)
    if variant is None:
        cmd = _nodes_command()
        if verbose:
            print(" ".join(cmd))
        procs.append(("row_autograd.cpp", subprocess.Popen(cmd)))
    for src in sources():
        obj = os.path.join(objdir, os.path.basename(src)[:-4] + ".o")
        objs.append(obj)
        cmd = [hipcc, f"--offload-arch={ARCH}", *FLAGS, *extra_flags, "-I", os.path.join(ROOT, "include"), "-I", HERE, "-c", src, "-o", obj]
        if verbose:
            print(" ".join(cmd))
        procs.append((src, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"compiler failed on {src}")
    cmd = [hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", lib, *objs]
    subprocess.run(cmd, check=True)
    return lib


if __name__ == "__main__":
    # python -m holoscene_amd.csrc.build [--force] [--variant NAME -DFLAG ...]
    args = sys.argv[1:]
    var = args[args.index("--variant") + 1] if "--variant" in args else None
    print(build(force="--force" in args, verbose=True, variant=var, extra_flags=[a for a in args if a.startswith("-D")]))
