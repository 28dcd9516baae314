"""build(): the C library does not wait for what calls it from torch (no compiler runs here)."""
import os
import sys

import pytest

from dynamis_amd import build


@pytest.fixture
def calls(monkeypatch, tmp_path):
    """build() in a folder of its own, with compilers that only write their output; what they were called with."""
    made = []

    def run(cmd):
        made.append(cmd)
        if cmd[0] == build.CXX:
            raise RuntimeError("no headers here")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(cmd))
        return ""

    for name, path in (("HERE", ""), ("LIB", "libdynamis_graph.so"), ("TORCH_LAYER", "_torch_layer.so")):
        monkeypatch.setattr(build, name, str(tmp_path / path))
    monkeypatch.setattr(build, "_run", run)
    return made


def test_the_library_is_linked_without_the_calls_from_torch(calls):
    with pytest.raises(RuntimeError, match="no headers here"):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.TORCH_LAYER)
    assert "-shared" in open(build.LIB).read()


def test_the_library_is_all_where_there_is_no_torch(calls, monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert all(cmd[0] != build.CXX for cmd in calls)


def test_a_source_that_fails_leaves_no_library(calls, monkeypatch):
    run = build._run
    monkeypatch.setattr(build, "_run", lambda cmd: (_ for _ in ()).throw(RuntimeError("bad source")) if "-c" in cmd else run(cmd))
    with pytest.raises(RuntimeError, match="bad source"):
        build.build()
    assert not os.path.exists(build.LIB)
