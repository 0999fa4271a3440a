"""The Python binding belongs to the torch and the Python that it was built for: another one rebuilds it, and does not run it."""
import os

import pytest

import stlq_b200
from stlq_b200 import build, operators

pytest.importorskip("torch")


@pytest.fixture
def commands(monkeypatch):
    """The build's commands, recorded and not run, and nothing else of it written."""
    run = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: run.append(cmd))
    return run


def test_another_torch_rebuilds_it(monkeypatch, tmp_path, commands):
    monkeypatch.setattr(build, "OBJDIR", str(tmp_path))
    monkeypatch.setattr(build, "BINDING_OUT", str(tmp_path / "_operators.so"))
    build.build_binding()
    assert len(commands) == 1 and any("STLQ_BUILT_FOR" in a for a in commands[0])
    (tmp_path / "_operators.so").write_text("")
    build.build_binding()
    assert len(commands) == 1  # nothing changed
    monkeypatch.setattr(build, "built_for", lambda: "torch 99.0, cpython-312")
    build.build_binding()
    assert len(commands) == 2 and any("torch 99.0" in a for a in commands[1])
    build.build_binding()
    assert len(commands) == 2


def test_one_built_for_another_torch_is_refused(monkeypatch):
    operators._ready()
    monkeypatch.setattr(operators, "_READY", None)
    monkeypatch.setattr(build, "built_for", lambda: "torch 99.0, cpython-312")
    with pytest.raises(stlq_b200.StlqB200Error, match="torch 99.0.*stlq_b200.build"):
        operators._ready()


def test_this_one_is_for_this_torch():
    import torch

    assert torch.__version__ in operators._ready()[1].BUILT_FOR and os.path.exists(build.BINDING_OUT)
