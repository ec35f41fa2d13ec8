"""What the build compiles, with the compilers stood in for."""
import importlib.util
import os

import pytest

from tcb_b200 import build as B


@pytest.fixture
def compiled(tmp_path, monkeypatch):
    """build() into an empty folder, its commands noted and their outputs made empty."""
    seen = []

    def run(cmd, check):
        out = cmd[cmd.index("-o") + 1]
        seen.append(os.path.basename(out))
        open(out, "w").close()

    monkeypatch.setattr(B, "HERE", str(tmp_path))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "libtcb.so"))
    monkeypatch.setattr(B, "TORCH_LIB", str(tmp_path / "_tcb_torch.so"))
    monkeypatch.setattr(B.subprocess, "run", run)
    # the C ABI's header is not beside that folder
    monkeypatch.setattr(B.os.path, "getmtime", lambda p, get=os.path.getmtime: get(p) if os.path.exists(p) else 0.0)

    def build(**kw):
        seen.clear()
        B.build(**kw)
        return list(seen)

    return build


def test_without_torch_the_library_is_built(compiled, monkeypatch):
    found = importlib.util.find_spec
    monkeypatch.setattr(B.importlib.util, "find_spec", lambda name, *a: None if name == "torch" else found(name, *a))
    made = compiled(force=True)
    assert "libtcb.so" in made and "tcb_serve.o" in made and "_tcb_torch.so" not in made


def test_the_torch_view_is_built_again_for_another_torch_or_python(compiled, monkeypatch):
    assert "_tcb_torch.so" in compiled(force=True)
    assert compiled() == []
    version = B.importlib.metadata.version
    monkeypatch.setattr(B.importlib.metadata, "version", lambda name: "99.0" if name == "torch" else version(name))
    assert compiled() == ["_tcb_torch.so"] and compiled() == []
    monkeypatch.setattr(B.sys, "version", "3.99")
    assert compiled() == ["_tcb_torch.so"] and compiled() == []
