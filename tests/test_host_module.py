"""The C++ host module belongs to the torch that it was compiled against (CPU test): another one builds it anew, and does not
load it as it is."""
import pytest
import torch

from erfnet_pytorch_amd import _lib


def compiled(monkeypatch):
    """The host module's compilations that build() asks for."""
    asked = []
    monkeypatch.setattr(_lib, "_run", lambda cmd, verbose: asked.append(cmd))
    _lib.build()
    return [c for c in asked if c[c.index("-o") + 1] == _lib._HOST_SO]


def test_the_module_says_which_torch_it_was_built_for(monkeypatch):
    _lib.host()
    assert _lib._host_built_for() == torch.__version__
    assert compiled(monkeypatch) == []


def test_another_torch_builds_it_anew(monkeypatch):
    _lib.host()
    monkeypatch.setattr(torch, "__version__", "1.2.3+other")
    cmd, = compiled(monkeypatch)
    assert '-DERF_TORCH_VERSION="1.2.3+other"' in cmd


def test_another_torch_does_not_load_it(monkeypatch):
    _lib.host()
    monkeypatch.setattr(torch, "__version__", "1.2.3+other")
    monkeypatch.setattr(_lib, "_host_module", None)
    with pytest.raises(RuntimeError, match="built for torch .* this is 1.2.3"):
        _lib.host()


def test_a_file_that_does_not_say_is_built_anew(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_HOST_SO", str(tmp_path / "_host.so"))
    assert _lib._host_built_for() is None and len(compiled(monkeypatch)) == 1
    (tmp_path / "_host.so").write_bytes(b"something else")
    assert _lib._host_built_for() is None and len(compiled(monkeypatch)) == 1
    monkeypatch.setattr(_lib, "_host_module", None)
    with pytest.raises(RuntimeError, match="does not say"):
        _lib.host()
