"""Builds ``libtir.so`` (the C-ABI library) in-tree for sm_100a.

Each source is compiled to an object under ``_build/`` (parallel, rebuilt only
when a source or header is newer), then linked with the static CUDA runtime so
the library loads on a machine without a GPU.
"""
import concurrent.futures
import glob
import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
CSRC = os.path.join(ROOT, "csrc")
INCLUDE = os.path.join(os.path.dirname(ROOT), "include")
BUILD = os.path.join(ROOT, "_build")
LIB = os.path.join(PKG_DIR, "libtir.so")
BIND_SRC = os.path.join(ROOT, "bind", "paged_bind.cpp")
BIND = os.path.join(PKG_DIR, "_paged_bind" + sysconfig.get_config_var("EXT_SUFFIX"))
BIND_STAMP = os.path.join(BUILD, "paged_bind.stamp")  # what BIND was compiled against

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O2,-ffp-contract=off",
              "--expt-relaxed-constexpr", "-I" + INCLUDE]


def nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build libtir.so")


def _sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cpp")))


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.cuh")) + \
        glob.glob(os.path.join(INCLUDE, "*.h"))


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, verbose):
    obj = os.path.join(BUILD, os.path.basename(src) + ".o")
    if not _stale(obj, [src, *_headers(), __file__]):
        return obj
    cmd = [nvcc(), *ARCH, *NVCC_FLAGS, "-c", src, "-o", obj]
    if src.endswith(".cu") and verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    if verbose and r.stderr:
        print(r.stderr, file=sys.stderr)
    return obj


def _bind_target():
    """The torch and Python a binding is good for; None without torch."""
    if importlib.util.find_spec("torch") is None:
        return None
    return f"torch {importlib.metadata.version('torch')}, {sysconfig.get_config_var('SOABI')}"


def build_bind():
    """Compiles the torch binding of the paged cache operators (needs torch's and
    Python's headers; without torch installed there are no tensors to bind)."""
    target = _bind_target()
    if target is None:
        return None
    if not _stale(BIND, [BIND_SRC, *_headers(), __file__]) and os.path.exists(BIND_STAMP):
        with open(BIND_STAMP) as f:
            if f.read() == target:
                return BIND
    os.makedirs(BUILD, exist_ok=True)
    import torch
    torch_dir = os.path.dirname(torch.__file__)
    inc = os.path.join(torch_dir, "include")
    lib = os.path.join(torch_dir, "lib")
    abi = int(getattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", True))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-w",
           f"-D_GLIBCXX_USE_CXX11_ABI={abi}", f'-DTIR_BIND_TORCH="{torch.__version__}"', "-I" + inc,
           "-I" + os.path.join(inc, "torch", "csrc", "api", "include"), "-I" + sysconfig.get_paths()["include"], BIND_SRC,
           "-o", BIND, "-L" + lib, "-Wl,-rpath," + lib, "-ltorch_python", "-ltorch_cpu", "-lc10"]
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{e}") from e
    if r.returncode != 0:
        raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
    with open(BIND_STAMP, "w") as f:
        f.write(target)
    return BIND


def build(verbose=False):
    """Compiles every CUDA/C++ source and links libtir.so; returns its path.  With
    torch installed its binding of the paged cache operators is compiled, too;
    nothing else needs that, so a failure there is only printed (build_bind()
    raises it, and the first call of such an operator says that it is missing)."""
    os.makedirs(BUILD, exist_ok=True)
    srcs = _sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs)) + 1) as ex:
        bind = ex.submit(build_bind)
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
        if _stale(LIB, objs):
            cmd = [nvcc(), *ARCH, "-shared", "-cudart", "static", "-o", LIB, *objs, "-lpthread", "-ldl", "-lrt"]
            r = subprocess.run(cmd, capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"link failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        try:
            bind.result()
        except Exception as e:
            print(f"{LIB} is built, the torch binding of the paged cache operators is not: {e}", file=sys.stderr)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
