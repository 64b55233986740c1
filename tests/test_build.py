"""CPU checks of the build's steps, without running them: what is built without torch, and when the torch binding is built again."""
import os
import sys

import pytest

from chpl_b200 import build as b


@pytest.fixture
def steps(monkeypatch, tmp_path):
    """The files that a build would write, in order; nothing is compiled, no file of the tree touched."""
    made = []

    def run(cmd, verbose):
        made.append(cmd[cmd.index("-o") + 1])

    monkeypatch.setattr(b, "_run", run)
    monkeypatch.setattr(b, "BUILD", str(tmp_path))
    return made


EXES = [os.path.join(b.BIN, name) for name in b.EXES]


def test_without_torch_everything_else_is_built(steps, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # `import torch` raises ImportError
    assert b.build(force=True) == b.LIB
    assert b.LIB in steps and all(e in steps for e in EXES) and b.TORCH_EXT not in steps
    assert "torch" in capsys.readouterr().err


def test_with_torch_the_binding_is_built_last(steps):
    b.build(force=True)
    assert b.LIB in steps and all(e in steps for e in EXES) and steps[-1] == b.TORCH_EXT


def test_another_torch_builds_the_binding_again(steps, monkeypatch):
    import torch
    b.build(force=True)
    monkeypatch.setattr(b, "_newer", lambda target, deps: False)
    steps.clear()
    b.build()
    assert steps == []
    monkeypatch.setattr(torch, "__version__", "0.0")
    b.build()
    assert steps == [b.TORCH_EXT]


def test_a_binding_that_does_not_compile_is_an_error(steps, monkeypatch):
    def fail(cmd, verbose):
        if b.TORCH_EXT in cmd:
            raise RuntimeError("build step failed")
        steps.append(cmd[cmd.index("-o") + 1])

    monkeypatch.setattr(b, "_run", fail)
    with pytest.raises(RuntimeError):
        b.build(force=True)
    assert all(e in steps for e in EXES)
