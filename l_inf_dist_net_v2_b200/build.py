"""Builds libldn_b200.so (sm_100a only) in-tree with nvcc.

    python l_inf_dist_net_v2_b200/build.py [--force] [--verbose]

(run it as a script: importing the package needs the library this script produces)

Each translation unit is compiled on its own (in parallel) and the objects are linked into
l_inf_dist_net_v2_b200/libldn_b200.so.  nvcc cross-compiles without a GPU.
"""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
OBJ = os.path.join(CSRC, "_obj")
LIB = os.path.join(PKG, "libldn_b200.so")

NVCC_FLAGS = [
    "-std=c++17", "-O3", "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo",
    "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", "-I", os.path.join(ROOT, "include"), "-I", CSRC,
]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cuh")]
    hs.append(os.path.join(ROOT, "include", "ldn_b200.h"))
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=False):
    os.makedirs(OBJ, exist_ok=True)
    headers = _headers()
    jobs = []
    objs = []
    for src in _sources():
        s = os.path.join(CSRC, src)
        o = os.path.join(OBJ, src[:-3] + ".o")
        objs.append(o)
        if force or _stale(o, [s] + headers):
            cmd = ["nvcc"] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o]
            jobs.append(cmd)

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        return cmd, r

    if jobs:
        with ThreadPoolExecutor(max_workers=min(len(jobs), os.cpu_count() or 4)) as ex:
            for cmd, r in ex.map(run, jobs):
                if verbose or r.returncode != 0:
                    sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
                if r.returncode != 0:
                    raise RuntimeError("nvcc failed for " + cmd[-3])
    if jobs or force or _stale(LIB, objs):
        cmd = ["nvcc", "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + objs
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(r.stdout + r.stderr)
            raise RuntimeError("link failed")
    return LIB


EXT_NAME = "_norm_dist_ext"
EXT_SRCS = [os.path.join(CSRC, "binding", f) for f in ("norm_dist_ext.cpp", "head_ext.cpp")]


def ext_path():
    import sysconfig
    return os.path.join(PKG, EXT_NAME + sysconfig.get_config_var("EXT_SUFFIX"))


def build_extension(force=False, verbose=False):
    """Compiles the pybind11 / PyTorch binding (csrc/binding/*.cpp) against libldn_b200.so, in-tree.
    Plain g++ with the include and library paths torch reports; no GPU needed."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension as ce
    out = ext_path()
    header = os.path.join(ROOT, "include", "ldn_b200.h")
    if not force and not _stale(out, EXT_SRCS + [header]):
        return out
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden",
           "-DTORCH_EXTENSION_NAME=" + EXT_NAME, "-DTORCH_API_INCLUDE_EXTENSION_H",
           "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch.compiled_with_cxx11_abi())]
    for inc in ce.include_paths() + [sysconfig.get_paths()["include"], os.path.join(cuda_home, "include"),
                                    os.path.join(ROOT, "include")]:
        cmd += ["-isystem" if "torch" in inc or "python" in inc else "-I", inc]
    os.makedirs(OBJ, exist_ok=True)
    objs = [os.path.join(OBJ, os.path.basename(s)[:-4] + ".ext.o") for s in EXT_SRCS]

    def run(cmd):
        return cmd, subprocess.run(cmd, capture_output=True, text=True)

    def checked(cmd, r):
        if verbose or r.returncode != 0:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
        if r.returncode != 0:
            raise RuntimeError("building the PyTorch binding failed")

    with ThreadPoolExecutor(max_workers=len(EXT_SRCS)) as ex:
        for c, r in ex.map(run, [cmd + ["-c", s, "-o", o] for s, o in zip(EXT_SRCS, objs) if force or _stale(o, [s, header])]):
            checked(c, r)
    checked(*run(["g++", "-shared"] + objs +
                 ["-o", out, "-L", torch_lib, "-L", PKG, "-lldn_b200", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda",
                  "-ltorch", "-ltorch_python", "-Wl,-rpath,$ORIGIN", "-Wl,-rpath," + torch_lib]))
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
    if "--no-ext" not in sys.argv:
        print(build_extension(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
