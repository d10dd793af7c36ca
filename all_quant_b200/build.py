"""Builds libuq_b200.so in-tree with nvcc for sm_100a (the only target), and the host module _uq_host.so.  Run as
`python -m all_quant_b200.build` or through __graft_entry__.build(); `--lib` builds the library alone, which needs neither torch nor Python's
headers (the C ABI; the Python entry points of the operators around the attention need the module as well)."""
import hashlib
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
OBJ = os.path.join(HERE, "build")
LIB = os.path.join(HERE, "libuq_b200.so")
HOST = os.path.join(HERE, "_uq_host.so")   # the Python module of csrc/uq_host.cpp (g++ against torch's headers)
STAMP = os.path.join(OBJ, "_uq_host.stamp")   # what HOST was built from, see _host_stamp
SOURCES = ["uq_api.cu", "uq_append.cu", "uq_verify_fma.cu", "uq_verify_tc.cu", "uq_combine.cu", "uq_layout.cu", "uq_plan.cu", "uq_rows.cu", "uq_linear.cu"]
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC",
         "-I", INCLUDE, "-I", CSRC] + os.environ.get("UQ_NVCC_EXTRA", "").split()


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _header_id():
    """The flag that gives the library and the host module the digest of the C ABI's header: each says which text it was built from."""
    with open(os.path.join(INCLUDE, "uq_b200.h"), "rb") as f:
        return "-DUQB_HEADER_ID=0x" + hashlib.sha256(f.read()).hexdigest()[:16] + "ull"


def _host_command():
    import sysconfig
    import torch
    t, cuda = os.path.dirname(torch.__file__), os.path.dirname(os.path.dirname(NVCC))
    inc = [os.path.join(t, "include"), os.path.join(t, "include", "torch", "csrc", "api", "include"), os.path.join(cuda, "include"), sysconfig.get_paths()["include"]]
    return (["g++", "-O2", "-std=c++17", "-fPIC", "-shared", os.path.join(CSRC, "uq_host.cpp"), "-o", HOST, f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
             f'-DUQ_TORCH_VERSION="{torch.__version__}"', _header_id(), "-I", INCLUDE]
            + [x for d in inc for x in ("-isystem", d)]
            + [f"-L{os.path.join(t, 'lib')}", "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python", f"-Wl,-rpath,{os.path.join(t, 'lib')}"])


def _host_stamp():
    """What the host module depends on besides its source: the C ABI's header, this interpreter and its torch (looked up without importing it)."""
    import importlib.metadata
    import importlib.util
    spec = importlib.util.find_spec("torch")
    return "\n".join([_header_id(), sys.version, spec.origin if spec else "no torch", importlib.metadata.version("torch") if spec else ""])


def _host_is_stale():
    if _stale(HOST, [os.path.join(CSRC, "uq_host.cpp")]) or not os.path.exists(STAMP):
        return True
    with open(STAMP) as f:
        return f.read() != _host_stamp()


def _run(cmd):
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError("the compiler failed: " + " ".join(cmd) + "\n" + r.stdout + r.stderr)
    return r.stderr


def _build_host():
    _run(_host_command())
    with open(STAMP, "w") as f:
        f.write(_host_stamp())


def build(force=False, verbose=False, host=True):
    """The library, then (host) the module: where the module cannot be built, the library is there all the same and the error says so."""
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".cuh", ".h"))]
    headers += [os.path.join(INCLUDE, f) for f in os.listdir(INCLUDE)]
    os.makedirs(OBJ, exist_ok=True)
    jobs = []
    for src in SOURCES:
        s, o = os.path.join(CSRC, src), os.path.join(OBJ, src + ".o")
        if force or _stale(o, [s] + headers):
            jobs.append([NVCC] + FLAGS + [_header_id()] + (["-Xptxas", "-v"] if verbose else []) + ["-c", s, "-o", o])

    with ThreadPoolExecutor(max_workers=4) as ex:
        module = ex.submit(_build_host) if host and (force or _host_is_stale()) else None
        for log in ex.map(_run, jobs):
            if verbose and log:
                print(log)
        objs = [os.path.join(OBJ, s + ".o") for s in SOURCES]
        if jobs or force or _stale(LIB, objs):
            _run([NVCC, "-shared", "-o", LIB] + objs + ["-gencode", "arch=compute_100a,code=sm_100a"])
        if module is not None:
            try:
                module.result()
            except Exception as e:
                raise RuntimeError(f"{LIB} is built, the host module {HOST} is not (build(host=False), --lib: the library alone)") from e
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv, host="--lib" not in sys.argv))
