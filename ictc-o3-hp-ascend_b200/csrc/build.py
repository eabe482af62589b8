"""Build libictc_cuda.so for sm_100a from the CUDA sources in this folder.

Each .cu file is compiled to an object in parallel, then linked into
``ictc_o3/backends/cuda/libictc_cuda.so`` beside the Python package that
loads it.  The CUDA runtime is linked statically, so the library carries no
dependency on a particular libcudart soname.  host_tensors.cpp becomes a Python
extension module beside it (g++, against the installed torch and this interpreter);
where that fails, the package runs without it.

    python build.py [--force] [--verbose]
"""
import argparse
import concurrent.futures
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
REPO = os.path.dirname(PKG)
INCLUDE = os.path.join(REPO, "include")
OBJDIR = os.path.join(PKG, "_build")
OUTPUT = os.path.join(PKG, "ictc_o3", "backends", "cuda", "libictc_cuda.so")
HOST_SOURCE = os.path.join(HERE, "host_tensors.cpp")
HOST_OUTPUT = os.path.join(PKG, "ictc_o3", "backends", "cuda", "_host_tensors" + sysconfig.get_config_var("EXT_SUFFIX"))
NVCC = os.environ.get("NVCC", "nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
         "-Xcompiler", "-fPIC", "-I" + INCLUDE, "-I" + HERE]


def sources():
    return sorted(f for f in os.listdir(HERE) if f.endswith(".cu"))


def _deps_mtime():
    stamps = [os.path.getmtime(os.path.join(HERE, f)) for f in os.listdir(HERE)
              if f.endswith((".cuh", ".h"))]
    stamps += [os.path.getmtime(os.path.join(INCLUDE, f)) for f in os.listdir(INCLUDE)]
    return max(stamps) if stamps else 0.0


def _compile(src, force, verbose):
    obj = os.path.join(OBJDIR, src[:-3] + ".o")
    path = os.path.join(HERE, src)
    if (not force and os.path.exists(obj)
            and os.path.getmtime(obj) >= max(os.path.getmtime(path), _deps_mtime())):
        return obj
    cmd = [NVCC, *FLAGS, "-c", path, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{proc.stderr}")
    if verbose:
        sys.stderr.write(proc.stderr)
    return obj


def build_host(force=False):
    """The extension module of host_tensors.cpp; without torch it has no user and is left out."""
    try:
        import torch
    except ImportError:
        return None
    root = os.path.dirname(os.path.abspath(torch.__file__))
    # times of installed files say nothing: an older torch may be installed later
    built_for, stamp = f"{torch.__version__}\n{root}\n", os.path.join(OBJDIR, "host_tensors.torch")
    if (not force and os.path.exists(HOST_OUTPUT) and os.path.exists(stamp) and open(stamp).read() == built_for
            and os.path.getmtime(HOST_OUTPUT) >= os.path.getmtime(HOST_SOURCE)):
        return HOST_OUTPUT
    tmp = HOST_OUTPUT + ".tmp"
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DICTC_TORCH_VERSION="{torch.__version__}"',
           "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
           "-I" + sysconfig.get_paths()["include"], HOST_SOURCE, "-L" + os.path.join(root, "lib"),
           "-lc10", "-ltorch_cpu", "-ltorch_python", "-o", tmp]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"g++ failed for host_tensors.cpp:\n{proc.stderr}")
    os.replace(tmp, HOST_OUTPUT)
    with open(stamp, "w") as f:
        f.write(built_for)
    return HOST_OUTPUT


def build(force=False, verbose=False):
    os.makedirs(OBJDIR, exist_ok=True)
    output = build_kernels(force, verbose)
    try:
        build_host(force)
    except (RuntimeError, OSError) as error:      # no g++, or no headers of Python or torch: slower, not unusable
        if os.path.exists(HOST_OUTPUT):
            os.remove(HOST_OUTPUT)
        sys.stderr.write(f"{error}\nwithout _host_tensors the optimizer reads its tensors' addresses in Python and "
                         "block norms refuse captured backward passes\n")
    return output


def build_kernels(force=False, verbose=False):
    srcs = sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=max(1, min(len(srcs), os.cpu_count() or 1))) as pool:
        objs = list(pool.map(lambda s: _compile(s, force, verbose), srcs))
    if (not force and os.path.exists(OUTPUT)
            and os.path.getmtime(OUTPUT) >= max(os.path.getmtime(o) for o in objs)):
        return OUTPUT
    tmp = OUTPUT + ".tmp"
    cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-cudart", "static",
           *objs, "-o", tmp]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed:\n{proc.stderr}")
    os.replace(tmp, OUTPUT)
    return OUTPUT


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    args = parser.parse_args()
    print(build(args.force, args.verbose))
