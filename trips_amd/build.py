"""Builds libtrips_splat.so (HIP kernels + C ABI) in-tree for gfx950 with hipcc."""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libtrips_splat.so")
SOURCES = ["trips_splat_abi.hip", "splat_forward.hip", "splat_backward.hip", "misc_kernels.hip", "unet_forward.hip",
           "unet_backward.hip", "adamw_kernels.hip", "lookup_kernels.hip", "loss_kernels.hip", "dropout_kernels.hip"]
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off",
    # packed FP32 instructions are kept out of the generated code on purpose
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function",
]


def hipcc():
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found")


HEADERS = ["splat_internal.h", "trips_math.h", "row16.h", "unet_common.h", "abi_common.h", os.path.join("..", "..", "include", "trips_splat.h"),
           os.path.join("..", "..", "include", "trips_unet.h"), os.path.join("..", "..", "include", "trips_optim.h"),
           os.path.join("..", "..", "include", "trips_lookup.h"), os.path.join("..", "..", "include", "trips_loss.h")]


def build(verbose=False, incremental=False):
    """One hipcc process per translation unit, side by side, then one link. `incremental` skips units whose object
    is newer than the unit and every header (a convenience while editing; the default compiles everything)."""
    objdir = os.path.join(CSRC, "_obj")
    os.makedirs(objdir, exist_ok=True)
    newest_header = max(os.path.getmtime(os.path.join(CSRC, h)) for h in HEADERS)
    procs, objs = [], []
    for src in SOURCES:
        path = os.path.join(CSRC, src)
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        objs.append(obj)
        if incremental and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(path), newest_header):
            continue
        cmd = [hipcc()] + FLAGS + ["-c", path, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((cmd, subprocess.Popen(cmd)))
    for cmd, pr in procs:
        if pr.wait() != 0:
            raise subprocess.CalledProcessError(pr.returncode, cmd)
    link = [hipcc(), "--offload-arch=gfx950", "-shared", "-fPIC"] + objs + ["-o", LIB]
    if verbose:
        print(" ".join(link), flush=True)
    subprocess.check_call(link)
    return LIB


SHIM_DIR = os.path.join(CSRC, "torch_shim")
SHIM_LIB = os.path.join(HERE, "_trips_torch.so")
HOST_LIB = os.path.join(HERE, "_trips_host.so")


def _has_torch():
    try:
        import torch  # noqa: F401
    except ImportError:
        return False
    return True


def _torch_flags(name):
    """(compiler flags, linker flags) of a libtorch extension that calls the C ABI of libtrips_splat.so."""
    import sysconfig

    import torch
    from torch.utils import cpp_extension as ce
    tlib = ce.library_paths()[0]
    inc = [f"-I{p}" for p in ce.include_paths()] + [f"-I{sysconfig.get_paths()['include']}", "-I/opt/rocm/include"]
    abi_flag = f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"
    flags = (["-O2", "-std=c++17", "-fPIC", "-Wall", "-Wno-unused-variable", abi_flag, "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
              f"-DTORCH_EXTENSION_NAME={name}", "-DTORCH_API_INCLUDE_EXTENSION_H"] + inc)
    return flags, [f"-L{tlib}", f"-L{HERE}", "-ltrips_splat", "-lc10", "-lc10_hip", "-ltorch_cpu", "-ltorch_hip", "-ltorch",
                   "-ltorch_python", f"-Wl,-rpath,{tlib}", "-Wl,-rpath,$ORIGIN"]


def _build_torch_extension(name, sources, lib, verbose, incremental=False):
    """Plain g++, one process per translation unit, side by side: these hold no device code."""
    flags, libs = _torch_flags(name)
    objdir = os.path.join(SHIM_DIR, "_obj")
    os.makedirs(objdir, exist_ok=True)
    include = os.path.join(HERE, "..", "include")
    headers = [os.path.join(d, f) for d in (SHIM_DIR, include) for f in os.listdir(d) if f.endswith(".h")]
    newest_header = max(os.path.getmtime(h) for h in headers)
    procs, objs = [], []
    for f in sources:
        path, obj = os.path.join(SHIM_DIR, f), os.path.join(objdir, f.replace(".cpp", ".o"))
        objs.append(obj)
        if incremental and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(path), newest_header):
            continue
        cmd = ["g++"] + flags + ["-c", path, "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((cmd, subprocess.Popen(cmd)))
    for cmd, pr in procs:
        if pr.wait() != 0:
            raise subprocess.CalledProcessError(pr.returncode, cmd)
    link = ["g++", "-shared"] + objs + libs + ["-o", lib]
    if verbose:
        print(" ".join(link), flush=True)
    subprocess.check_call(link)
    return lib


def build_host(verbose=False, incremental=False):
    """Builds _trips_host.so, the host side of trips_amd/adamw.py, lookup.py, table_loss.py and dropout.py; after build(), whose library it links."""
    return _build_torch_extension("_trips_host", ("trips_host.cpp",), HOST_LIB, verbose, incremental)


def build_torch_shim(verbose=False):
    """Builds the libtorch host side (PointRender / NeuralRenderInfo / MyAdam in C++) with a pybind11 test driver."""
    sources = ("trips_torch.cpp", "trips_unet_torch.cpp", "trips_scene_io.cpp", "trips_torch_py.cpp")
    return _build_torch_extension("_trips_torch", sources, SHIM_LIB, verbose)


if __name__ == "__main__":
    build(verbose=True, incremental="--incremental" in sys.argv)
    print(LIB)
    if _has_torch():
        print(build_host(verbose=True, incremental="--incremental" in sys.argv))
    else:
        print("no torch: _trips_host.so, which adamw.py, lookup.py, table_loss.py and dropout.py need, is left out")
    if "--shim" in sys.argv:
        print(build_torch_shim(verbose=True))
