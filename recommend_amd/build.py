"""Build librecommend_amd.so (gfx950) in-tree with hipcc.

The library is the C-ABI declared in include/recommend_amd.h; it is built here
on a CPU-only host (hipcc cross-compiles) and travels to the GPU box as a file.
Beside it _torch_ops.so, a Python module of host code (g++).
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "librecommend_amd.so")
SOURCES = ["host.cpp", "graph.hip", "spmm.hip", "dense.hip", "dense_wide.hip", "glue.hip", "optim.hip", "bpr.hip", "eval.hip", "eval_filter.hip", "knn.hip", "proj.hip",
           "embedding.hip", "preference.hip", "adamw.hip"]
FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-fno-fast-math", "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    # no v_pk_{add,mul,fma}_f32: some of their forms have given wrong results on this hardware now and
    # then (hipcc's host pass does not know the feature and says so: harmless)
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-function", "-Wno-inline-asm",
]


# the operators' torch side (argument checks, buffers, autograd nodes): host code against torch's own headers
TORCH_OPS = "torch_ops.cpp"
TORCH_OPS_PATH = os.path.join(LIB_DIR, "_torch_ops.so")


def torch_ops_command(out):
    import sysconfig

    import torch
    root = os.path.dirname(torch.__file__)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-unused-function", "-D__HIP_PLATFORM_AMD__=1",
            "-DUSE_ROCM", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-I" + os.path.join(root, "include"), "-I" + os.path.join(root, "include", "torch", "csrc", "api", "include"),
            "-I" + sysconfig.get_paths()["include"], "-I" + os.path.join(rocm, "include"),
            os.path.join(CSRC, TORCH_OPS), "-o", out, "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_hip", "-ltorch_cpu",
            "-ltorch_python"]


def _stale(path, sources):
    """Whether `path` is missing or older than one of `sources`, the header or this file."""
    if not os.path.exists(path):
        return True
    deps = [os.path.join(CSRC, f) for f in sources] + [os.path.join(HERE, "..", "include", "recommend_amd.h"),
                                                       os.path.abspath(__file__)]
    return any(os.path.getmtime(d) > os.path.getmtime(path) for d in deps)


def needs_library():
    return _stale(LIB_PATH, [f for f in os.listdir(CSRC) if f != TORCH_OPS])


def needs_torch_ops():
    return _stale(TORCH_OPS_PATH, [TORCH_OPS])


def needs_build():
    return needs_library() or needs_torch_ops()


def build(force=False, verbose=True):
    """The library needs hipcc alone; it is complete where the torch module, compiled beside it, fails (which raises)."""
    library, module = force or needs_library(), force or needs_torch_ops()
    os.makedirs(LIB_DIR, exist_ok=True)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

    def start(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        return subprocess.Popen(cmd)

    torch_ops = None
    if module:
        # (never one of other sources beside the library: it relies on the header's signatures)
        if os.path.exists(TORCH_OPS_PATH):
            os.remove(TORCH_OPS_PATH)
        try:
            torch_ops = start(torch_ops_command(TORCH_OPS_PATH))
        except (ImportError, OSError) as e:
            print(e, file=sys.stderr)
    if library:
        objs = [os.path.join(LIB_DIR, src + ".o") for src in SOURCES]
        procs = [start([hipcc, "-x", "hip"] + [f for f in FLAGS if f != "-shared"] + ["-c", os.path.join(CSRC, src), "-o", obj])
                 for src, obj in zip(SOURCES, objs)]
        failed = [src for src, p in zip(SOURCES, procs) if p.wait() != 0]
        if failed:
            raise RuntimeError(f"the compiler failed on {', '.join(failed)}")
        if start([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs).wait() != 0:
            raise RuntimeError("linking the library failed")
    if module and (torch_ops is None or torch_ops.wait() != 0):
        raise RuntimeError(f"the compiler failed on {TORCH_OPS}: the library is complete, but embedding_lookup, list_logps, "
                           "preference_loss and FusedAdamW will not run")
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB_PATH)
