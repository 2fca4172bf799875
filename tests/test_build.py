"""CPU: the build of the native library does not depend on the torch extension's."""

import importlib.metadata
import sys
import types

import pytest

from easy_as_b200 import build


@pytest.mark.parametrize("torch", ["fails to import", "lacks what the build asks for", "is absent"])
def test_the_library_is_built_beside_a_torch_that(torch, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build, "needs_build", lambda: False)
    monkeypatch.setattr(build, "OPS", tmp_path / "eas_ops.so")
    monkeypatch.setattr(build, "OPS_STAMP", tmp_path / "eas_ops.so.sha256")
    if torch == "is absent":
        def version(name):
            raise importlib.metadata.PackageNotFoundError(name)

        monkeypatch.setattr(importlib.metadata, "version", version)
    else:
        module = None if torch == "fails to import" else types.ModuleType("torch")
        if module is not None:
            module.__file__ = str(tmp_path / "torch" / "__init__.py")
            module._C = types.SimpleNamespace()
        monkeypatch.setitem(sys.modules, "torch", module)
    assert build.build() == build.LIB
    assert not (tmp_path / "eas_ops.so").exists()
    assert ("not built" in capsys.readouterr().err) == (torch != "is absent")
