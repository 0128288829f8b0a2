"""Build libcpmcu_b200.so in-tree with nvcc for sm_100a, and the Python module _ops.so over it with g++ against torch's headers.

Usage: python cpm.cu_b200/build.py [--force]
Both land next to the Python package (cpm.cu_b200/cpmcu/) so that they
travel with the source tree; nothing is installed into site-packages.  The library is built first and
stands alone: what goes wrong with the module, or a machine without torch, does not touch it.
"""
import concurrent.futures
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
OUT_DIR = os.path.join(HERE, "cpmcu")
OBJ_DIR = os.path.join(HERE, "build")
LIB = os.path.join(OUT_DIR, "libcpmcu_b200.so")
OPS = os.path.join(OUT_DIR, "_ops.so")   # Python module over the library, for torch tensors
SOURCES = ["runtime.cu", "gemm_umma.cu", "gemm_pair.cu", "gemm_w4_umma.cu", "elementwise.cu", "tree_attn.cu", "pair_attn.cu", "draft_tree.cu", "accept.cu",
           "marlin_unpack.cu", "sparse_select.cu", "sparse_stage1.cu", "layered_ops.cu", "plain_ops.cu", "one_row.cu", "tanh_rows.cu", "recurrence.cu", "moe.cu", "engine.cu", "engine_layered.cu", "w8a8_rows.cu", "w8a8_one_row.cu", "gemm_w8a8.cu", "rotary.cu", "op_errors.cu", "capi_ops.cu", "capi.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "-Xcompiler", "-fPIC", "--threads", "2"]
# extra defines for instrumented builds, e.g. CPMCU_BUILD_DEFINES="-DCPMCU_W4_PROFILE=1"
NVCC_FLAGS += os.environ.get("CPMCU_BUILD_DEFINES", "").split()


def _nvcc():
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if cand and (os.path.isabs(cand) and os.path.exists(cand) or not os.path.isabs(cand)):
            return cand
    return "nvcc"


def _hash(files, *words):
    h = hashlib.sha256()
    for path in files:
        with open(path, "rb") as f:
            h.update(os.path.basename(path).encode())
            h.update(f.read())
    h.update(" ".join(words).encode())
    return h.hexdigest()


def _sources(*endings):
    return [os.path.join(root, name) for root in (CSRC, os.path.join(os.path.dirname(HERE), "include")) for name in sorted(os.listdir(root)) if name.endswith(endings)]


def _stamp():
    return _hash(_sources(".cu", ".cuh", ".h"), *NVCC_FLAGS)


def _ops_stamp(command):
    """Of the module: its source, the header of the library, and the torch and Python that it is compiled for."""
    import torch
    return _hash(_sources(".cpp", ".h"), torch.__version__, sys.version, *command)


def _fresh(output, stamp_file, stamp):
    if not (os.path.exists(output) and os.path.exists(stamp_file)):
        return False
    with open(stamp_file) as f:
        return f.read() == stamp


def _run(cmd, what):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("%s:\n%s\n%s" % (what, res.stdout, res.stderr))


def _write(path, text):
    with open(path, "w") as f:
        f.write(text)


def _forget(stamp_file):
    """Before a build: one that ends half-way leaves nothing that counts as built."""
    if os.path.exists(stamp_file):
        os.remove(stamp_file)


def _ops_command(cuda_home):
    """g++ command that compiles csrc/torch_ops.cpp and links it against the library beside it and torch's own libraries."""
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch._C._GLIBCXX_USE_CXX11_ABI),
           os.path.join(CSRC, "torch_ops.cpp"), "-o", OPS]
    cmd += ["-isystem" + d for d in (os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"),
                                     os.path.join(cuda_home, "include"), sysconfig.get_paths()["include"])]
    return cmd + ["-L" + OUT_DIR, "-l:libcpmcu_b200.so", "-Wl,-rpath,$ORIGIN", "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
                  "-ltorch_python"]


def build_library(force=False, verbose=True):
    """libcpmcu_b200.so: nvcc alone."""
    os.makedirs(OBJ_DIR, exist_ok=True)
    stamp_file, stamp = os.path.join(OBJ_DIR, "stamp"), _stamp()
    if not force and _fresh(LIB, stamp_file, stamp):
        return LIB
    _forget(stamp_file)
    nvcc = _nvcc()

    def compile_one(src):
        obj = os.path.join(OBJ_DIR, src.replace(".cu", ".o"))
        _run([nvcc] + NVCC_FLAGS + ["-c", os.path.join(CSRC, src), "-o", obj], "nvcc failed for %s" % src)
        return obj

    with concurrent.futures.ThreadPoolExecutor(max_workers=4) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    _run([nvcc, "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a", "-lcudart"], "link failed")
    _write(stamp_file, stamp)
    if verbose:
        print("built", LIB)
    return LIB


def build_module(force=False, verbose=True):
    """_ops.so over the library, with g++ against torch's headers; None where there is no torch: the library and its C entry points stand without it."""
    try:
        import torch  # noqa: F401
    except ImportError:
        print("no torch: %s is not built, and cpmcu.w8a8 and cpmcu.rotary cannot be imported" % os.path.basename(OPS))
        return None
    os.makedirs(OBJ_DIR, exist_ok=True)
    nvcc = _nvcc()
    command = _ops_command(os.path.dirname(os.path.dirname(nvcc)) if os.path.isabs(nvcc) else "/usr/local/cuda")
    stamp_file, stamp = os.path.join(OBJ_DIR, "stamp_ops"), _ops_stamp(command)
    if not force and _fresh(OPS, stamp_file, stamp):
        return OPS
    _forget(stamp_file)
    _run(command, "g++ failed for torch_ops.cpp")
    _write(stamp_file, stamp)
    if verbose:
        print("built", OPS)
    return OPS


def build(force=False, verbose=True):
    build_library(force, verbose)
    build_module(force, verbose)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
