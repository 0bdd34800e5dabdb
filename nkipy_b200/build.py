"""Build ``libnkb.so`` (the C-ABI runtime + kernel library) and ``nkb_torch.so`` in-tree.

Every ``csrc/*.cu`` file is compiled for sm_100a only
(``-gencode arch=compute_100a,code=sm_100a``) with ``nvcc`` and linked into
``nkipy_b200/_lib/libnkb.so``.  ``csrc/torch_serving.cpp``, the serving calls on
torch tensors, becomes the Python module ``_lib/nkb_torch.so`` against the
installed torch's headers, where that torch has CUDA.  Objects are rebuilt when
their source or a header is newer, the module also for another torch or Python.
Run ``python -m nkipy_b200.build``.
"""

import concurrent.futures
import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "_lib")
OBJ_DIR = os.path.join(HERE, "_lib", "obj")
LIB = os.path.join(OUT_DIR, "libnkb.so")
TORCH_LIB = os.path.join(OUT_DIR, "nkb_torch.so")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")

NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CUDA_INCLUDE = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "-Xcompiler",
    "-fvisibility=hidden",
    "--expt-relaxed-constexpr",
    f"-I{INCLUDE}",
]


def _sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _headers():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    hs += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE) if f.endswith(".h")]
    return hs


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, verbose):
    obj = os.path.join(OBJ_DIR, os.path.basename(src).replace(".cu", ".o"))
    if not _stale(obj, [src] + _headers()):
        return obj
    cmd = [NVCC] + FLAGS + ["-c", src, "-o", obj]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{r.stdout}\n{r.stderr}")
    return obj


def built_for(torch_version, torch_git):
    """What the module's binary interface goes with, besides its sources."""
    return f"torch {torch_version} {torch_git}, {sys.implementation.cache_tag}"


def _installed(torch):
    """``built_for`` of the torch package in a folder, by its record of its own build."""
    record = {}
    with open(os.path.join(torch, "version.py")) as f:
        exec(f.read(), {"__name__": "torch.version"}, record)
    return built_for(record["__version__"], record.get("git_version"))


def _build_torch(verbose):
    """Build ``nkb_torch.so``; None where there is no torch with CUDA to build it against,
    which libnkb.so does without (the calls that need the module then say that it is missing)."""
    spec = importlib.util.find_spec("torch")
    if spec is None or not spec.submodule_search_locations:
        return None
    torch = spec.submodule_search_locations[0]
    if not os.path.exists(os.path.join(torch, "lib", "libc10_cuda.so")):
        print("nkb_torch.so is not built: the installed torch has no CUDA libraries", file=sys.stderr)
        return None
    src, record, goes_with = os.path.join(CSRC, "torch_serving.cpp"), os.path.join(OBJ_DIR, "nkb_torch.built"), _installed(torch)
    known = None
    if os.path.exists(record):
        with open(record) as f:
            known = f.read()
    if known == goes_with and not _stale(TORCH_LIB, [src, os.path.join(INCLUDE, "nkb.h")]):
        return TORCH_LIB
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared", src, "-o", TORCH_LIB, f'-DNKB_BUILT_FOR="{goes_with}"']
    cmd += [f"-I{d}" for d in (INCLUDE, os.path.join(torch, "include"), os.path.join(torch, "include/torch/csrc/api/include"),
                               sysconfig.get_paths()["include"], CUDA_INCLUDE)]
    cmd += [f"-L{OUT_DIR}", "-lnkb", f"-L{os.path.join(torch, 'lib')}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed for {src}:\n{r.stdout}\n{r.stderr}")
    with open(record, "w") as f:
        f.write(goes_with)
    return TORCH_LIB


def build(verbose=False) -> str:
    os.makedirs(OBJ_DIR, exist_ok=True)
    srcs = _sources()
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    if _stale(LIB, objs):
        cmd = [NVCC, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", LIB] + objs + ["-lcuda", "-ldl"]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    _build_torch(verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
