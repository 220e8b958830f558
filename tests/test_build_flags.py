"""An object is rebuilt when the command that made it is not the one that would make
it now: sources and headers alone would keep code of other flags."""
import subprocess
import types
from pathlib import Path

import pytest

from hipdsml import _build


@pytest.fixture
def fake(monkeypatch, tmp_path):
    """The build with its compiler and linker replaced by file writes."""
    made = []

    def run(cmd, **_):
        out = Path(cmd[cmd.index("-o") + 1])
        out.write_text("")
        made.append(out.name)
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(_build, "OBJ", tmp_path / "build" / "obj")
    monkeypatch.setattr(_build, "OUT", tmp_path / "_C.so")
    monkeypatch.setattr(subprocess, "run", run)

    def build(**kw):
        made.clear()
        _build.build(**kw)
        return set(made)

    return build


def test_objects_of_other_flags_are_rebuilt(fake, monkeypatch):
    everything = fake()
    assert "_C.so" in everything and "route.hip.o" in everything and "bindings_experts.o" in everything
    assert fake() == set()
    monkeypatch.setattr(_build, "ARCH", "gfx000")
    changed = fake()
    # the device code and the link know the architecture, the bindings do not
    assert changed == {o for o in everything if not o.startswith("bindings")}
    assert fake() == set()
    monkeypatch.setattr(_build, "CSRC", _build.CSRC / "." / ".." / "csrc")  # another include path in every command
    assert fake() == everything


def test_objects_without_a_record_are_rebuilt(fake):
    """A directory that an earlier build left, whatever its flags were."""
    everything = fake()
    for record in _build.OBJ.glob("*.cmd"):
        record.unlink()
    assert fake() == everything
    (_build.OBJ / "route.hip.o.cmd").write_text("hipcc -O0")
    assert fake() == {"route.hip.o", "_C.so"}


def test_a_failed_compile_leaves_no_record(fake, monkeypatch):
    fake()
    monkeypatch.setattr(_build, "ARCH", "gfx000")
    good = subprocess.run

    def fail(cmd, **kw):
        if "route" in cmd[-1]:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no")
        return good(cmd, **kw)

    monkeypatch.setattr(subprocess, "run", fail)
    with pytest.raises(RuntimeError, match="compile failed"):
        fake()
    monkeypatch.setattr(subprocess, "run", good)
    assert "route.hip.o" in fake()
