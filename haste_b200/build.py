"""Build recipe: compile the CUDA sources under csrc/ for sm_100a and link libhaste_ffi.so in-tree, and beside it the Python
extension ``_dense`` through which torch tensors reach the dense operators.

    python -m haste_b200.build            # incremental (skips objects newer than their sources)
    python -m haste_b200.build --force

nvcc cross-compiles without a GPU.  The library links the CUDA runtime statically and depends on
nothing else (no torch, no Python).  The extension is host code alone, built against the installed torch, and again when that is another.
"""
import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libhaste_ffi.so")
DENSE = os.path.join(HERE, "_dense" + sysconfig.get_config_var("EXT_SUFFIX"))
SOURCES = ["api.cu", "runtime.cu", "ffi_mma.cu", "ffi_step_sm100_g128.cu", "ffi_step_sm100_g64.cu", "ffi_step_sm100_small.cu", "ffi_forward_sm100.cu", "ffi_backward_sm100.cu", "elementwise.cu", "rewire.cu", "topk.cu", "layernorm.cu", "adamw.cu", "probes.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
              "--expt-relaxed-constexpr", "-Xptxas", "-v"]


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    raise RuntimeError("nvcc not found")


def _newest_header():
    hs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".cuh"))]
    hs.append(os.path.join(HERE, "..", "include", "haste_ffi.h"))
    return max(os.path.getmtime(h) for h in hs)


def _compile(src, force):
    obj = os.path.join(OBJ, src.replace(".cu", ".o"))
    srcp = os.path.join(CSRC, src)
    if (not force and os.path.exists(obj) and os.path.getmtime(obj) > os.path.getmtime(srcp)
            and os.path.getmtime(obj) > _newest_header()):
        return obj, ""
    cmd = [_nvcc()] + NVCC_FLAGS + ["-c", srcp, "-o", obj]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"nvcc failed for {src}:\n{p.stdout}\n{p.stderr}")
    return obj, p.stderr


def _build_dense(force):
    src = os.path.join(CSRC, "dense_binding.cpp")
    newest = max(os.path.getmtime(src), os.path.getmtime(os.path.join(HERE, "..", "include", "haste_ffi.h")))
    import torch
    from torch.utils import cpp_extension
    stamp, against = os.path.join(OBJ, "_dense.torch"), f"{torch.__version__} {torch.__file__}"
    if not force and os.path.exists(DENSE) and os.path.getmtime(DENSE) > newest and os.path.exists(stamp):
        with open(stamp) as f:
            if f.read() == against:
                return
    made = os.path.join(OBJ, os.path.basename(DENSE))
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
    for path in cpp_extension.include_paths() + [sysconfig.get_path("include"), os.path.join(os.path.dirname(os.path.dirname(_nvcc())), "include")]:
        cmd += ["-isystem", path]
    cmd += [src, "-o", made]
    for path in cpp_extension.library_paths():
        cmd += ["-L" + path]
    cmd += ["-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    p = subprocess.run(cmd, capture_output=True, text=True)
    if p.returncode != 0:
        raise RuntimeError(f"compiling dense_binding.cpp failed:\n{p.stdout}\n{p.stderr}")
    os.replace(made, DENSE)
    with open(stamp, "w") as f:
        f.write(against)


def build(force=False, verbose=False):
    os.makedirs(OBJ, exist_ok=True)
    with ThreadPoolExecutor(max_workers=len(SOURCES) + 1) as ex:
        dense = ex.submit(_build_dense, force)
        results = list(ex.map(lambda s: _compile(s, force), SOURCES))
    objs = [o for o, _ in results]
    log = "".join(l for _, l in results)
    if log:
        with open(os.path.join(OBJ, "ptxas.log"), "w") as f:
            f.write(log)
    if verbose and log:
        print(log)
    if force or not os.path.exists(LIB) or any(os.path.getmtime(o) > os.path.getmtime(LIB) for o in objs):
        cmd = [_nvcc(), "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a"]
        p = subprocess.run(cmd, capture_output=True, text=True)
        if p.returncode != 0:
            raise RuntimeError(f"link failed:\n{p.stdout}\n{p.stderr}")
    dense.result()                                      # without the extension there is the library, which needs none of it
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
