"""The build's two products, no GPU and no compiler needed: the plugin asks for no torch, the binding is built for the
torch that is there."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from libr3d_b200 import build, ops

ROOT = Path(__file__).resolve().parent.parent
NO_TORCH = ("import sys, runpy; sys.path.insert(0, %r); sys.modules['torch'] = None\n"
            "from libr3d_b200 import build\nbuild._stale = lambda *a: False\n" % str(ROOT))


def _run(code):
    return subprocess.run([sys.executable, "-c", NO_TORCH + code], capture_output=True, text=True, env=os.environ | {"PYTHONWARNINGS": "ignore"})


def test_the_plugin_is_built_without_torch():
    r = _run("print(build.build_plugin())")
    assert r.returncode == 0 and r.stdout.strip() == str(build.SO), r.stderr


def test_the_command_says_that_the_binding_is_left_out():
    r = _run("main = open(build.__file__).read().split('if __name__')[1].split(':', 1)[1]\nexec('if True:' + main, vars(build))")
    assert r.returncode == 0 and "torch is not installed" in r.stderr and r.stdout.split() == [str(build.SO)], r.stderr


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    ran = []

    class Done:
        returncode = 0

    monkeypatch.setattr(build, "_stale", lambda *a: False)
    monkeypatch.setattr(build, "BIND_FOR", tmp_path / "bind_for.txt", raising=False)
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or Done)
    build.build_bind()
    assert len(ran) == 1                              # nothing says what the file that is there was built against
    build.build_bind()
    assert len(ran) == 1
    monkeypatch.setattr(torch, "__version__", "0.0")
    build.build_bind()
    assert len(ran) == 2


@pytest.mark.parametrize("there,word", [(True, "does not load with this torch"), (False, "is not built")])
def test_a_binding_that_does_not_load_says_why(monkeypatch, plug, there, word):
    import libr3d_b200
    ops.plugin()
    monkeypatch.setitem(sys.modules, "libr3d_b200._bind", None)
    monkeypatch.delattr(libr3d_b200, "_bind", raising=False)
    monkeypatch.setattr(ops, "_bind", None)
    if not there:
        monkeypatch.setattr(ops.Path, "exists", lambda self: False)
    with pytest.raises(ImportError, match=word):
        ops._load_bind()
