"""Builds libuq_b200.so in-tree with nvcc for sm_100a (the only target), and the host module _uq_host.so.  Run as
`python -m all_quant_b200.build` or through __graft_entry__.build()."""
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libuq_b200.so")
HOST = os.path.join(HERE, "_uq_host.so")   # the Python module of csrc/uq_host.cpp (g++ against torch's headers)
SOURCES = ["uq_api.cu", "uq_append.cu", "uq_verify_fma.cu", "uq_verify_tc.cu", "uq_combine.cu", "uq_layout.cu", "uq_plan.cu", "uq_rows.cu", "uq_linear.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
         "-I", os.path.join(ROOT, "include"), "-I", CSRC] + os.environ.get("UQ_NVCC_EXTRA", "").split()


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _host_command():
    import sysconfig
    import torch
    t, cuda = os.path.dirname(torch.__file__), os.path.dirname(os.path.dirname(NVCC))
    inc = [os.path.join(t, "include"), os.path.join(t, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", os.path.join(CSRC, "uq_host.cpp"), "-o", HOST, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}"]
            + [x for d in inc for x in ("-isystem", d)]
            + [f"-L{os.path.join(t, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", f"-Wl,-rpath,{os.path.join(t, 'lib')}"])


def build(force=False, verbose=False):
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers += [os.path.join(ROOT, "include", f) for f in os.listdir(os.path.join(ROOT, "include"))]
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    jobs = []
    for src in SOURCES:
        s, o = os.path.join(CSRC, src), os.path.join(objdir, src + ".o")
        if force or _stale(o, [s] + headers):
            jobs.append([NVCC] + FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o])

    cuda_jobs = len(jobs)
    if force or _stale(HOST, [os.path.join(CSRC, "uq_host.cpp")]):
        jobs.append(_host_command())

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("the compiler failed: " + " ".join(cmd) + "\n" + r.stdout + r.stderr)
        return r.stderr

    with ThreadPoolExecutor(max_workers=4) as ex:
        for log in ex.map(run, jobs):
            if verbose and log:
                print(log)
    objs = [os.path.join(objdir, s + ".o") for s in SOURCES]
    if cuda_jobs or force or _stale(LIB, objs):
        run([NVCC, "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a"])
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
