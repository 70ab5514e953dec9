"""Building in places that lack a part."""

import sys

from tosa_b200 import build as B


def test_without_torch_the_library_is_built_alone(monkeypatch, tmp_path, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    monkeypatch.setattr(B, "BINDING", str(tmp_path / "_torch_binding.so"))
    assert B.build() == B.OUT
    assert "torch is not installed" in capsys.readouterr().err
    assert not (tmp_path / "_torch_binding.so").exists()
