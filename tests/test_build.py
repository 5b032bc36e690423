"""What build() makes, with the compilers stood in for (no GPU)."""
import sys

import pytest

from ishizuki_amd import build


@pytest.mark.parametrize("torch_there", [True, False])
def test_the_library_needs_no_torch(monkeypatch, torch_there, tmp_path, capsys):
    """Without torch the C library is built all the same, and its Python binding left out."""
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(build, "BIND", str(tmp_path / "bind.so"))
    monkeypatch.setattr(build, "_compile", lambda src: src + ".o")

    def run(cmd, **_):
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Done", (), {"returncode": 0})
    monkeypatch.setattr(build.subprocess, "run", run)
    if not torch_there:
        for name in ("torch", "torch.utils"):
            monkeypatch.setitem(sys.modules, name, None)
    assert build.build() == str(tmp_path / "lib.so")
    assert (tmp_path / "lib.so").exists() and (tmp_path / "bind.so").exists() == torch_there
    assert ("no torch" in capsys.readouterr().out) == (not torch_there)
