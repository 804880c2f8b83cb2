"""Build the in-tree CUDA library libexactb200.so for sm_100a (nvcc, no torch dependency) and, beside it,
libexactb200_torch.so (g++ and torch's headers): the torch operators that call it (torch_ops.cpp).

Every .cu file compiles to its own object in parallel (whole-program device code per file, no
relocatable device code: the translation units share only inline header code), then one nvcc
call links the shared library."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
SRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(ROOT, "_build")
LIB = os.path.join(HERE, "libexactb200.so")
TORCH_SRC = os.path.join(HERE, "torch_ops.cpp")
TORCH_LIB = os.path.join(HERE, "libexactb200_torch.so")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-Wall",
         "--expt-relaxed-constexpr", "-I", os.path.join(ROOT, "include"), "-I", SRC]
LIBS = ["-ldl"]                       # NCCL (tensor parallelism) is opened at run time


def sources():
    return sorted(os.path.join(SRC, f) for f in os.listdir(SRC) if f.endswith(".cu"))


def headers():
    hs = [os.path.join(SRC, f) for f in os.listdir(SRC) if f.endswith((".cuh", ".h"))]
    return hs + [os.path.join(ROOT, "include", "exactb200.h")]


def needs_build():
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    return any(os.path.getmtime(p) > t for p in sources() + headers())


def _obj(src):
    return os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")


def build(force=False, verbose=False, extra=()):
    if not force and not needs_build():
        return LIB
    os.makedirs(OBJ, exist_ok=True)
    newest_header = max(os.path.getmtime(p) for p in headers())
    flags = ARCH + FLAGS + list(extra)

    def compile_one(src):
        o = _obj(src)
        if (not force and os.path.exists(o) and os.path.getmtime(o) > os.path.getmtime(src)
                and os.path.getmtime(o) > newest_header and not extra):
            return None
        cmd = [NVCC] + flags + ["-c", "-o", o + ".tmp", src]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            return f"{src}:\n{r.stdout}{r.stderr}"
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)
        os.replace(o + ".tmp", o)
        return None

    with ThreadPoolExecutor(max_workers=max(1, min(len(sources()), os.cpu_count() or 4))) as ex:
        errs = [e for e in ex.map(compile_one, sources()) if e]
    if errs:
        raise RuntimeError("nvcc failed:\n" + "\n".join(errs))
    cmd = [NVCC] + ARCH + ["-shared", "-o", LIB + ".tmp"] + [_obj(s) for s in sources()] + LIBS
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(LIB + ".tmp", LIB)
    return LIB


def build_torch(force=False, verbose=False):
    """The torch operators.  Needs torch; without it there is nothing to register them with."""
    try:
        import torch
        from torch.utils.cpp_extension import include_paths, library_paths
    except ImportError:
        print("torch is not installed: no torch operators")
        return None
    newest = max(os.path.getmtime(p) for p in (TORCH_SRC, os.path.join(ROOT, "include", "exactb200.h")))
    made_for = f"{torch.__version__} {os.path.dirname(torch.__file__)}"       # the library fits this torch alone
    stamp = os.path.join(OBJ, "torch_ops.torch")
    if not force and os.path.exists(TORCH_LIB) and os.path.getmtime(TORCH_LIB) > newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == made_for:
                return TORCH_LIB
    import sysconfig
    cuda = os.path.dirname(os.path.dirname(NVCC))
    inc = include_paths() + [sysconfig.get_paths()["include"], os.path.join(cuda, "include"), os.path.join(ROOT, "include")]
    libs = library_paths()
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-unknown-pragmas",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}", "-DTORCH_API_INCLUDE_EXTENSION_H",
           "-o", TORCH_LIB + ".tmp", TORCH_SRC]
    cmd += [x for i in inc for x in ("-isystem", i)]
    cmd += [f"-L{d}" for d in libs] + ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    cmd += [f"-Wl,-rpath,{d}" for d in libs]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(TORCH_LIB + ".tmp", TORCH_LIB)
    os.makedirs(OBJ, exist_ok=True)
    with open(stamp, "w") as f:
        f.write(made_for)
    return TORCH_LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, extra=[a for a in sys.argv[1:] if a != "--force"])
    build_torch(force="--force" in sys.argv, verbose=True)
