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


# A library from before the training operators: the entries it has answer, the others are missing.
OLD = """
const char* sinkslot_last_error(void) { return ""; }
int sinkslot_abi_version(void) { return %d; }
"""

# Compilers that put the libraries built before in their place (what is compiled is not at issue).
NVCC = """#!/bin/sh
out=; for a in "$@"; do [ "$prev" = -o ] && out=$a; prev=$a; done
case " $* " in *" -shared "*) cp "{built}" "$out";; *) : > "$out";; esac
"""
GXX = """#!/bin/sh
out=; for a in "$@"; do [ "$prev" = -o ] && out=$a; prev=$a; done
cp "{built}" "$out"
"""


def _script(path, text):
    path.write_text(text)
    path.chmod(0o755)


def _old_library(copy, abi):
    lib = copy / "sinkslot_b200" / LIB
    lib.unlink()
    source = copy / "old.c"
    source.write_text(OLD % abi)
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(lib), str(source)], check=True)
    return lib


def _age(copy, name):
    """As a pull of newer sources leaves it: the library is older than they are."""
    os.utime(copy / "sinkslot_b200" / name, (1_000_000_000, 1_000_000_000))


def _compilers(copy):
    tools = copy / "tools"
    tools.mkdir()
    _script(tools / "nvcc", NVCC.format(built=os.path.join(PACKAGE, LIB)))
    _script(tools / "g++", GXX.format(built=os.path.join(PACKAGE, TORCH_LIB)))
    return {"NVCC": str(tools / "nvcc"), "PATH": f"{tools}{os.pathsep}{os.environ['PATH']}"}


@pytest.mark.parametrize("abi,newer", [(101, True), (102, False)])
def test_a_library_from_other_sources_is_refused_where_it_is_used(copy, abi, newer):
    """Importing the package does not fail, with a stale library or one whose date is newer than the
    sources'; using it does, and says what to do."""
    _old_library(copy, abi)
    if not newer:
        _age(copy, LIB)
    out = _python(copy, USE + """
import sinkslot_b200 as sk
for call in (sk.load_library, lambda: use(sk)):
    try:
        call()
    except ImportError as e:
        print("raised", e)
""")
    assert out.count("raised") == 2 and out.count("sinkslot_b200.build") == 2


def test_build_over_a_library_from_other_sources(copy):
    """Built over, in the process that imported the package: what is loaded then is the new one."""
    _old_library(copy, 101)
    _age(copy, LIB)
    tools = _compilers(copy)
    out = _python(copy, USE + """
import sinkslot_b200 as sk
from sinkslot_b200 import build
build.build()
assert sk.load_library().sinkslot_abi_version() >= 102
print(*use(sk))
""", **tools)
    assert out.split() == ["5", "3"]


def test_build_command_runs_over_a_library_from_other_sources(copy):
    _old_library(copy, 101)
    _age(copy, LIB)
    r = subprocess.run([sys.executable, "-m", "sinkslot_b200.build"], cwd=copy,
                       env={**os.environ, "PYTHONPATH": str(copy), **_compilers(copy)},
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert (copy / "sinkslot_b200" / LIB).stat().st_size > 1 << 20


def test_built_libraries_register_on_import(copy):
    """Libraries of these sources: the operators are there once the package is imported.  A build
    that replaces a library that is loaded says that this process keeps the old one."""
    out = _python(copy, """
import os, warnings
import torch, sinkslot_b200
from sinkslot_b200 import build
print(torch.ops.sinkslot_b200.lookup.default._schema.name)
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    build.build()
print(*[w.message for w in seen if "new process" in str(w.message)])
""", **_compilers(copy))
    assert "sinkslot_b200::lookup" in out and "new process" in out


def test_build_gives_the_solver_where_the_bindings_do_not_compile(copy):
    """The solver's library is built and loads; the bindings of other sources are taken away, and
    the build command fails."""
    env = _compilers(copy)
    tools = copy / "tools"
    _age(copy, TORCH_LIB)
    _script(tools / "g++", "#!/bin/sh\necho no torch headers >&2\nexit 1\n")
    out = _python(copy, USE + """
import os, warnings
import sinkslot_b200 as sk
from sinkslot_b200 import build
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    assert build.build() == sk.LIB_PATH
print(*[w.message for w in seen])
assert sk.load_library().sinkslot_abi_version() >= 102
assert not os.path.exists(build.TORCH_LIB)
try:
    use(sk)
except ImportError as e:
    print("raised", e)
""", **env)
    assert "training operators" in out and "raised" in out
    r = subprocess.run([sys.executable, "-m", "sinkslot_b200.build"], cwd=copy,
                       env={**os.environ, "PYTHONPATH": str(copy), **env}, capture_output=True,
                       text=True, timeout=300)
    assert r.returncode != 0 and "no torch headers" in r.stderr
