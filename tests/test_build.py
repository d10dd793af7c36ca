"""What the build does around the compilers (none of which runs here), and what keeps the library and the host module of one build together."""
import ctypes
import os
import subprocess
import types

import pytest

from all_quant_b200 import build as b
from all_quant_b200 import uq_cuda


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    """Commands are recorded; `fail` names a program that answers with an error."""
    ran, fail = [], set()

    def run(cmd, **kw):
        ran.append(cmd)
        return types.SimpleNamespace(returncode=int(os.path.basename(cmd[0]) in fail), stdout="", stderr="no such header")
    monkeypatch.setattr(subprocess, "run", run)
    for name in ("OBJ", "LIB", "HOST", "STAMP"):
        monkeypatch.setattr(b, name, str(tmp_path / name))
    return ran, fail


def test_a_host_module_that_cannot_be_built_leaves_the_library(compilers):
    ran, fail = compilers
    fail.add("g++")
    with pytest.raises(RuntimeError, match="the host module .* is not"):
        b.build()
    assert [c for c in ran if c[:3] == [b.NVCC, "-shared", "-o"]] and sum("-c" in c for c in ran) == len(b.SOURCES)
    assert not os.path.exists(b.STAMP)   # tried again the next time


def test_the_library_alone_needs_no_torch(compilers, monkeypatch):
    ran, fail = compilers
    monkeypatch.setattr(b, "_host_command", lambda: pytest.fail("the host module was asked for"))
    monkeypatch.setattr(b, "_host_stamp", lambda: pytest.fail("the host module was asked for"))
    assert b.build(host=False) == b.LIB and ran and all(c[0] == b.NVCC for c in ran)


def test_the_host_module_follows_the_header_and_torch(compilers, monkeypatch):
    ran, fail = compilers
    for name in ("HOST", "LIB"):
        open(getattr(b, name), "w").close()
    b._build_host()
    assert not b._host_is_stale()
    with monkeypatch.context() as m:
        m.setattr(b, "_header_id", lambda: "-DUQB_HEADER_ID=0x1ull")
        assert b._host_is_stale()
    with monkeypatch.context() as m:
        m.setattr("importlib.metadata.version", lambda name: "0.0")
        assert b._host_is_stale()
    assert not b._host_is_stale()
    # both are told the header they are built from
    assert b._header_id() in b._host_command()
    b.build(force=True, host=False)
    assert all(b._header_id() in c for c in ran if "-c" in c)


def test_the_host_module_refuses_a_library_of_another_header():
    host = uq_cuda._host()
    at = [ctypes.cast(getattr(uq_cuda.lib(), f), ctypes.c_void_p).value for f in uq_cuda._HOST_FNS]
    assert uq_cuda.lib().uqb_header_id() == int(b._header_id().split("0x")[1][:16], 16) != 0
    other = ctypes.CFUNCTYPE(ctypes.c_ulonglong)(lambda: 5)
    with pytest.raises(RuntimeError, match="different builds"):
        host.bind(*at[:-1], ctypes.cast(other, ctypes.c_void_p).value)
    host.bind(*at)


def test_a_host_module_for_another_torch_is_refused(monkeypatch):
    import torch
    monkeypatch.setattr(uq_cuda, "_host_module", None)
    monkeypatch.setattr(torch, "__version__", "0.0")
    with pytest.raises(RuntimeError, match="was built for torch"):
        uq_cuda._host()
