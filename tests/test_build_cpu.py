"""The library's build does not depend on that of the autograd nodes."""
import ctypes
import os

import pytest

from muon_sr_amd import _build


@pytest.fixture
def small(tmp_path, monkeypatch):
    """A library of one source, and nodes of an earlier build, in a folder of their own."""
    source = tmp_path / "one.hip"
    source.write_text('extern "C" int one(void) { return 1; }\n')
    monkeypatch.setattr(_build, "HERE", str(tmp_path))
    monkeypatch.setattr(_build, "LIB", str(tmp_path / "libone.so"))
    monkeypatch.setattr(_build, "NODES", str(tmp_path / "_nodes.so"))
    monkeypatch.setattr(_build, "sources", lambda: [str(source)])
    (tmp_path / "_nodes.so").write_text("of an earlier library")
    return monkeypatch


def commands(compile_, link=("true",)):
    def of(obj, out):
        open(out, "w").write("new")
        return list(compile_), list(link)
    return of


def no_headers(obj, out):
    raise ImportError("no headers")


@pytest.mark.parametrize("nodes,named", [(commands(["false"]), "false failed"), (commands(["true"], ["false"]), "false failed"),
                                         (commands(["/no/such/compiler"]), "/no/such/compiler"), (no_headers, "no headers")],
                         ids=["compiler fails", "linker fails", "no compiler", "no headers"])
def test_nodes_that_cannot_be_built(small, nodes, named):
    """The library is linked, the error names what failed, and no nodes of an earlier library are left beside it."""
    small.setattr(_build, "nodes_commands", nodes)
    with pytest.raises(RuntimeError, match=named):
        _build.build()
    assert ctypes.CDLL(_build.LIB).one() == 1
    assert not os.path.exists(_build.NODES)


def test_both(small):
    small.setattr(_build, "nodes_commands", commands(["true"]))
    assert _build.build() == _build.LIB
    assert ctypes.CDLL(_build.LIB).one() == 1 and open(_build.NODES).read() == "new"
    # a source that does not compile leaves what is there
    open(_build.sources()[0], "w").write("no C++")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        _build.build()
    assert os.path.exists(_build.LIB) and os.path.exists(_build.NODES)
