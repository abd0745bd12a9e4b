"""The build links objects of the tree that it is run in, whatever the files'
times, and finds out an extension that lacks what the package calls."""
import os
import shutil
import subprocess
import sys

import pytest

from flodl_b200 import _ext

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MODULE = """
#include <Python.h>
#include "values.h"
int other();
static PyModuleDef def = {PyModuleDef_HEAD_INIT, "%(name)s", 0, -1, 0};
PyMODINIT_FUNC PyInit_%(name)s(void) {
  PyObject* m = PyModule_Create(&def);
  PyModule_AddIntConstant(m, "header", FROM_HEADER);
  PyModule_AddIntConstant(m, "other", %(other)s);
  return m;
}
"""


def lay_out(tree, version, when):
    """A package with the repository's build script, all of its files as old as `when`."""
    csrc = os.path.join(tree, "flodl_b200", "csrc")
    for d in ("bind", "runtime"):
        os.makedirs(os.path.join(csrc, d), exist_ok=True)
    shutil.copy(os.path.join(ROOT, "setup.py"), tree)
    files = {"__init__.py": "", "csrc/values.h": f"#define FROM_HEADER {version}\n",
             "csrc/bind/module.cpp": MODULE % dict(name="_C", other="other()"),
             "csrc/bind/other.cpp": f"int other() {{ return {version}; }}\n",
             "csrc/runtime/module.cpp": MODULE % dict(name="_native", other="0")}
    for name, text in files.items():
        path = os.path.join(tree, "flodl_b200", name)
        with open(path, "w") as f:
            f.write(text)
        os.utime(path, (when, when))


def build(tree, objects):
    env = {**os.environ, "MAX_JOBS": "4"}
    r = subprocess.run([sys.executable, "setup.py", "build_ext", "--inplace", "-t", objects], cwd=tree,
                       env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    code = "import flodl_b200._C as c, flodl_b200._native as n; print(c.header, c.other, n.header)"
    out = subprocess.run([sys.executable, "-c", code], cwd=tree, capture_output=True, text=True, timeout=60)
    return out.stdout.split()


def object_times(objects):
    return {os.path.join(d, f): os.stat(os.path.join(d, f)).st_mtime_ns
            for d, _, files in os.walk(objects) for f in files if f.endswith(".o")}


def test_build_of_another_version_at_one_path(tmp_path):
    """A tree whose files are older than another version's objects at its path."""
    tree, objects = str(tmp_path / "tree"), str(tmp_path / "objects")
    os.makedirs(tree)
    lay_out(tree, 1, 1_600_000_000)
    assert build(tree, objects) == ["1", "1", "1"]
    lay_out(tree, 2, 1_600_000_100)
    assert build(tree, objects) == ["2", "2", "2"]
    before = object_times(objects)
    assert len(before) == 3
    assert build(tree, objects) == ["2", "2", "2"]
    assert object_times(objects) == before  # an unchanged tree's objects are reused


class WithoutTwo:
    """`real` without two of its names."""
    __name__ = "flodl_b200._C"

    def __init__(self, real):
        self._real = real

    def __getattr__(self, name):
        if name in ("cross_attention", "qk_norm_rope"):
            raise AttributeError(name)
        return getattr(self._real, name)


def test_names_that_an_extension_lacks(monkeypatch):
    if _ext._C is None or _ext._native is None:
        pytest.skip("extensions are not built")
    assert _ext.missing_names() == []

    real = _ext._C
    monkeypatch.setattr(_ext, "cuda_ext", lambda: WithoutTwo(real))
    missing = {m.split(" ")[0] for m in _ext.missing_names()}
    assert missing == {"flodl_b200._C.cross_attention", "flodl_b200._C.qk_norm_rope"}
