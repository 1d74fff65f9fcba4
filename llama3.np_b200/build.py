"""Builds libllama3_b200.so in-tree with nvcc for sm_100a (no JIT cache: the .so must travel
with the repo snapshot to the GPU box).  `python llama3.np_b200/build.py [--force]`."""
import hashlib
import os
import subprocess
import sys
import warnings
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libllama3_b200.so")
TORCH_OPS = os.path.join(HERE, "_torch_ops.so")  # of every variant
TORCH_OPS_STAMP = os.path.join(OBJ, "torch_ops.stamp")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-std=c++17",
         "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-DL3_BUILD"]


def _sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _digest():
    h = hashlib.sha256(" ".join(FLAGS).encode())
    for root in (CSRC, os.path.join(os.path.dirname(HERE), "include")):
        for f in sorted(os.listdir(root)):
            if f.endswith((".cu", ".cuh", ".h")):
                h.update(f.encode())
                with open(os.path.join(root, f), "rb") as fh:
                    h.update(fh.read())
    return h.hexdigest()


def _made_from(stamp, dig):
    if not os.path.exists(stamp):
        return False
    with open(stamp) as f:
        return f.read() == dig


def _torch_folder():
    import importlib.util
    spec = importlib.util.find_spec("torch")
    return None if spec is None else list(spec.submodule_search_locations)[0]


def _torch_with_cuda():
    """torch's folder; None where torch is not installed, or without CUDA."""
    torch = _torch_folder()
    return torch if torch and os.path.exists(os.path.join(torch, "lib", "libc10_cuda.so")) else None


def _torch_ops_digest(torch):
    """What _torch_ops.so was made from: its source, the library's header, torch's version and Python's."""
    import sysconfig
    h = hashlib.sha256(str(sysconfig.get_config_var("SOABI")).encode())
    for path in (os.path.join(CSRC, "torch_ops.cpp"), os.path.join(os.path.dirname(HERE), "include", "llama3_b200.h"), os.path.join(torch, "version.py")):
        with open(path, "rb") as fh:
            h.update(fh.read())
    return h.hexdigest()


def _torch_ops(force=False):
    """_torch_ops.so: the operators on device buffers as calls on torch tensors (csrc/torch_ops.cpp).  The library itself does without
    torch: where that is not installed, or without CUDA, there is nothing to build, and where the extension cannot be built there is a warning
    and no file (paged.py and beam.py raise then)."""
    import sysconfig
    torch = _torch_with_cuda()
    if torch is None:
        return
    stamp, dig = TORCH_OPS_STAMP, _torch_ops_digest(torch)
    if not force and os.path.exists(TORCH_OPS) and _made_from(stamp, dig):
        return
    cuda = os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")
    inc = [os.path.join(torch, "include"), os.path.join(torch, "include", "torch", "csrc", "api", "include"), cuda, sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", os.path.join(CSRC, "torch_ops.cpp"), "-o", TORCH_OPS, *("-I" + i for i in inc),
           "-L" + os.path.join(torch, "lib"), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    for old in (TORCH_OPS, stamp):
        if os.path.exists(old):
            os.remove(old)
    try:
        r = subprocess.run(cmd, capture_output=True, text=True)
        failed = f"{r.stdout}\n{r.stderr}" if r.returncode != 0 else ""
    except OSError as e:
        failed = str(e)
    if failed:
        warnings.warn(f"the operators on torch tensors are not available: g++ failed on torch_ops.cpp:\n{failed}", RuntimeWarning, stacklevel=3)
        return
    os.makedirs(os.path.dirname(stamp), exist_ok=True)
    with open(stamp, "w") as f:
        f.write(dig)


def build(force: bool = False, verbose: bool = False, variant: str = "", defines=()) -> str:
    """`variant` + `defines` (e.g. "redux", ["-DL3_TC_ARGMAX_REDUX"]) build libllama3_b200_<variant>.so beside
    the default library from the same sources (selected at run time with L3_LIB_VARIANT=<variant>)."""
    global OBJ, LIB, FLAGS
    if variant:
        OBJ = os.path.join(HERE, "build_" + variant)
        LIB = os.path.join(HERE, f"libllama3_b200_{variant}.so")
        FLAGS = FLAGS + list(defines)
    os.makedirs(OBJ, exist_ok=True)
    _library(force, verbose)
    _torch_ops(force)
    return LIB


def _library(force, verbose):
    stamp = os.path.join(OBJ, "stamp")
    dig = _digest()
    if not force and os.path.exists(LIB) and _made_from(stamp, dig):
        return
    if not os.path.exists(NVCC):
        raise RuntimeError(f"nvcc not found at {NVCC}; libllama3_b200.so cannot be built here")

    def compile_one(src):
        obj = os.path.join(OBJ, src[:-3] + ".o")
        cmd = [NVCC, *FLAGS, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src}:\n{r.stdout}\n{r.stderr}")
        if verbose:
            sys.stderr.write(r.stderr)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        objs = list(ex.map(compile_one, _sources()))
    cmd = [NVCC, "-shared", "-o", LIB, *objs, "-gencode", "arch=compute_100a,code=sm_100a",
           "-cudart", "static", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    with open(stamp, "w") as f:
        f.write(dig)


if __name__ == "__main__":
    name = sys.argv[sys.argv.index("--variant") + 1] if "--variant" in sys.argv else ""
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, variant=name,
                defines=[a for a in sys.argv[1:] if a.startswith("-D")]))
