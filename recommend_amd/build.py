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


def needs_build():
    if not os.path.exists(LIB_PATH) or not os.path.exists(TORCH_OPS_PATH):
        return True
    t = min(os.path.getmtime(LIB_PATH), os.path.getmtime(TORCH_OPS_PATH))
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)]
    deps.append(os.path.join(HERE, "..", "include", "recommend_amd.h"))
    deps.append(os.path.abspath(__file__))
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    if not force and not needs_build():
        return LIB_PATH
    os.makedirs(LIB_DIR, exist_ok=True)
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    objs = []
    procs = []
    for src in SOURCES:
        obj = os.path.join(LIB_DIR, src + ".o")
        cmd = [hipcc, "-x", "hip"] + [f for f in FLAGS if f != "-shared"] + \
              ["-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, subprocess.Popen(cmd)))
        objs.append(obj)
    cmd = torch_ops_command(TORCH_OPS_PATH)
    if verbose:
        print(" ".join(cmd), flush=True)
    procs.append((TORCH_OPS, subprocess.Popen(cmd)))
    for src, p in procs:
        if p.wait() != 0:
            raise RuntimeError(f"the compiler failed on {src}")
    cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    return LIB_PATH


if __name__ == "__main__":
    build(force="--force" in sys.argv)
    print(LIB_PATH)
