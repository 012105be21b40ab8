"""The module behind the serving calls: built for the torch and from the sources that are
there, once, however many threads make the first call."""
import os
import shutil
import sys
import threading
import time

import pytest
import torch

from heteromm_b200 import build as B
from heteromm_b200 import serve


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """The sources in a place of their own, and a compiler that writes its command."""
    pkg, inc = tmp_path / "pkg", tmp_path / "include"
    (pkg / "src" / "py").mkdir(parents=True)
    inc.mkdir()
    shutil.copy(os.path.join(B.PKG, "src", "py", "serve_calls.cpp"), pkg / "src" / "py")
    shutil.copy(os.path.join(B.INC, "heteromm_cuda.h"), inc)
    runs = []

    def run(cmd):
        runs.append(cmd)
        time.sleep(0.05)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(cmd))

    monkeypatch.setattr(B, "PKG", str(pkg))
    monkeypatch.setattr(B, "INC", str(inc))
    monkeypatch.setattr(B, "LIB_DIR", str(pkg / "lib"))
    monkeypatch.setattr(B, "_run", run)
    return pkg, inc, runs


def test_built_once_and_again_for_other_sources_or_torch(tree, monkeypatch):
    pkg, inc, runs = tree
    first = B.build_serve_calls()
    assert os.listdir(pkg / "lib") == [os.path.basename(first)] and B.build_serve_calls() == first and len(runs) == 1
    os.utime(inc / "heteromm_cuda.h")                 # the same text, later
    assert B.build_serve_calls() == first and len(runs) == 1
    with open(inc / "heteromm_cuda.h", "a") as f:
        f.write("/* another */\n")
    second = B.build_serve_calls()
    assert second != first and len(runs) == 2 and os.listdir(pkg / "lib") == [os.path.basename(second)]
    with open(pkg / "src" / "py" / "serve_calls.cpp", "a") as f:
        f.write("// another\n")
    third = B.build_serve_calls()
    assert third != second and len(runs) == 3
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    other = B.build_serve_calls()
    assert other != third and len(runs) == 4 and os.path.exists(third)      # (that torch may still want it)


def test_a_failed_build_leaves_nothing(tree, monkeypatch):
    pkg, _, _ = tree

    def run(cmd):
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("half")
        raise RuntimeError("build failed")

    monkeypatch.setattr(B, "_run", run)
    with pytest.raises(RuntimeError):
        B.build_serve_calls()
    assert os.listdir(pkg / "lib") == []


def test_two_builds_at_once(tree):
    pkg, _, runs = tree
    out = []
    threads = [threading.Thread(target=lambda: out.append(B.build_serve_calls())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(set(out)) == 1 and len({c[c.index("-o") + 1] for c in runs}) == len(runs)     # no two write one file
    assert os.listdir(pkg / "lib") == [os.path.basename(out[0])]


def test_without_headers_the_rest_is_built(tree, monkeypatch, tmp_path):
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "nowhere" / "__init__.py"))
    assert not os.path.exists(B.LIB_DIR)
    assert B.build_serve_calls() == "" and tree[2] == []
    with pytest.raises(RuntimeError, match="headers"):
        serve._Calls().attention
    monkeypatch.setitem(sys.modules, "torch", None)   # import torch fails
    assert B.build_serve_calls() == ""


def test_without_sources_what_was_built_is_taken(tree):
    pkg, inc, runs = tree
    out = B.build_serve_calls()
    os.remove(inc / "heteromm_cuda.h")
    assert B.build_serve_calls() == out and len(runs) == 1
    os.remove(out)
    assert B.build_serve_calls() == "" and len(runs) == 1


def test_threads_that_call_first(monkeypatch):
    """One of them builds and loads; all get the same functions."""
    path, asked = B.build_serve_calls(), []

    def build():
        asked.append(threading.get_ident())
        time.sleep(0.05)
        return path

    monkeypatch.setattr(B, "build_serve_calls", build)
    calls, got = serve._Calls(), []
    threads = [threading.Thread(target=lambda: got.append(calls.grow)) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(asked) == 1 and len(got) == 8 and len({id(f) for f in got}) == 1
    with pytest.raises(AttributeError):
        calls.something
