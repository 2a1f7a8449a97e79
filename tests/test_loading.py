"""Which libraries are loaded when, without a GPU: copies of the package with a library missing, from
other sources or not loadable, each in a process of its own."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

PACKAGE = os.path.join(ROOT, "sinkslot_b200")
LIB, TORCH_LIB = "libsinkslot_b200.so", "libsinkslot_b200_torch.so"


@pytest.fixture(scope="module")
def built():
    from sinkslot_b200 import build
    build.build()


@pytest.fixture
def copy(built, tmp_path):
    """The package and its built libraries in a folder of their own."""
    for part in ("sinkslot_b200", "include"):
        shutil.copytree(os.path.join(ROOT, part), tmp_path / part,
                        ignore=shutil.ignore_patterns("__pycache__", "_build"))
    return tmp_path


def _python(where, code, **env):
    r = subprocess.run([sys.executable, "-W", "error::RuntimeWarning", "-c", code], cwd=where,
                       env={**os.environ, "PYTHONPATH": str(where), **env},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


USE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
def use(sk):
    with FakeTensorMode():
        return sk.embedding_lookup(torch.empty(4, 3, device="cuda"),
                                   torch.zeros(5, dtype=torch.int64, device="cuda")).shape
"""


@pytest.mark.parametrize("how", ["missing", "not loadable"])
def test_solver_library_loads_without_the_training_operators(copy, how):
    """load_library() gives the solver's library; the training operators say what they miss."""
    torch_lib = copy / "sinkslot_b200" / TORCH_LIB
    torch_lib.unlink()
    if how == "not loadable":
        torch_lib.write_bytes(b"not a library")
    out = _python(copy, USE + """
import sinkslot_b200 as sk
assert sk.load_library().sinkslot_abi_version() >= 102
try:
    use(sk)
except ImportError as e:
    print("raised", e)
""")
    assert "raised" in out and "sinkslot_b200.build" in out
