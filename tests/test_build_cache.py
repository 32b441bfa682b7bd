"""The build keeps objects between runs: a compile that ended half-way, one whose
source changed meanwhile and two builds at once leave nothing wrong behind.
nvcc is a stand-in that copies its source."""
import importlib.util
import os
import stat
import subprocess
import sys
import textwrap

import pytest

BUILD = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "my-inference-engine_b200", "build.py")

NVCC = """#!{python}
import os, sys, time
args = sys.argv[1:]
out = args[args.index("-o") + 1]
here = os.path.dirname(os.path.abspath(__file__))
with open(os.path.join(here, "trace"), "a") as f:
    f.write("begin %d %s\\n" % (os.getpid(), "link" if "-shared" in args else "compile"))
if "-shared" in args:
    data = "".join(open(a).read() for a in args if a.endswith(".o"))
else:
    data = open(args[args.index("-c") + 1]).read()
if os.path.exists(os.path.join(here, "die")):
    open(out, "w").write(data[:2])
    os._exit(9)
edit = os.path.join(here, "edit")
if os.path.exists(edit) and "-c" in args:
    os.remove(edit)
    time.sleep(0.05)
    open(args[args.index("-c") + 1], "w").write("edited")
    time.sleep(0.05)
time.sleep(0.05)
open(out, "w").write(data)
with open(os.path.join(here, "trace"), "a") as f:
    f.write("end %d\\n" % os.getpid())
"""


def _module(root):
    spec = importlib.util.spec_from_file_location("qmv_build_under_test", BUILD)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.PKG_DIR, m.REPO_DIR, m.CSRC, m.OBJ_DIR = root, root, root, os.path.join(root, "build")
    m.LIB_PATH = os.path.join(root, "lib.so")
    m.SOURCES, m.HEADERS, m.PUBLIC_HEADERS = ["a.cu", "b.cpp"], [], []
    m._nvcc = lambda: os.path.join(root, "nvcc")
    return m


@pytest.fixture
def root(tmp_path):
    nvcc = tmp_path / "nvcc"
    nvcc.write_text(NVCC.replace("{python}", sys.executable))
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    (tmp_path / "a.cu").write_text("first a")
    (tmp_path / "b.cpp").write_text(" and b")
    return str(tmp_path)


def _library(root):
    with open(os.path.join(root, "lib.so")) as f:
        return f.read()


def _write(root, name, text):
    with open(os.path.join(root, name), "w") as f:
        f.write(text)


def test_a_compile_that_died_is_done_again(root):
    m = _module(root)
    m.build_library()
    assert _library(root) == "first a and b"
    _write(root, "a.cu", "second a")
    _write(root, "die", "")
    with pytest.raises(RuntimeError):
        m.build_library()
    assert _library(root) == "first a and b"
    os.remove(os.path.join(root, "die"))
    m.build_library()
    assert _library(root) == "second a and b"


def test_a_source_that_changed_while_it_was_compiled_is_compiled_again(root):
    m = _module(root)
    m.SOURCES = ["a.cu"]
    _write(root, "edit", "")
    m.build_library()
    m.build_library()
    assert _library(root) == "edited"


def test_two_builds_at_once(root):
    """One waits for the other and finds the library there."""
    code = textwrap.dedent("""
        import sys
        sys.path.insert(0, %r)
        import test_build_cache
        test_build_cache._module(%r).build_library()
        """) % (os.path.dirname(os.path.abspath(__file__)), root)
    builds = [subprocess.Popen([sys.executable, "-c", code], stderr=subprocess.PIPE) for _ in range(3)]
    for b in builds:
        assert b.wait(60) == 0, b.stderr.read()
        b.stderr.close()
    assert _library(root) == "first a and b"
    with open(os.path.join(root, "trace")) as f:
        assert sum(line.startswith("begin") for line in f) == 3  # two sources, one link
    left = os.listdir(root) + os.listdir(os.path.join(root, "build"))
    assert not [f for f in left if ".tmp" in f], left
