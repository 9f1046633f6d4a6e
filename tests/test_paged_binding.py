"""The compiled binding of the paged entry points: when it is loaded, and that a build without
it is whole."""
import hashlib
import types
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parent.parent


def test_the_library_says_which_header_it_is_of(fl):
    want = hashlib.sha256((REPO / "include" / "fl355.h").read_bytes()).hexdigest()[:16]
    assert fl._lib.lib().fl_header_digest().decode() == want


def test_a_binding_of_another_build_is_not_bound(fl, monkeypatch):
    """Another header's or another torch's binding is declined with a warning, before it is
    given any address (the stand-in library has none to give)."""
    L = fl._lib.lib()
    assert fl._lib._load_binding(L) is not None
    other = types.SimpleNamespace(fl_header_digest=lambda: b"0123456789abcdef")
    with pytest.warns(RuntimeWarning, match="build again"):
        assert fl._lib._load_binding(other) is None
    same = types.SimpleNamespace(fl_header_digest=L.fl_header_digest)
    monkeypatch.setattr(torch, "__version__", "1.0")
    with pytest.warns(RuntimeWarning, match="build again"):
        assert fl._lib._load_binding(same) is None


def test_a_binding_that_does_not_say_what_it_is_of_is_not_bound(fl, monkeypatch):
    """One from before bindings said so."""
    module = types.SimpleNamespace()
    monkeypatch.setattr(fl._lib.importlib.util, "module_from_spec", lambda spec: module)
    monkeypatch.setattr(fl._lib.importlib.machinery.ExtensionFileLoader, "exec_module", lambda self, m: None)
    with pytest.warns(RuntimeWarning, match="build again"):
        assert fl._lib._load_binding(fl._lib.lib()) is None


def test_a_build_without_a_cxx_compiler_has_no_binding(fl, monkeypatch, tmp_path, capsys):
    """The binding is optional: its build says so and takes an old one away, and the loader
    takes its absence."""
    import __graft_entry__ as ge
    builder = ge._load_builder()
    old = tmp_path / "fl355_paged.so"
    old.write_bytes(b"of an earlier build")
    monkeypatch.setattr(builder, "BINDING_PATH", old)
    monkeypatch.setattr(builder.shutil, "which", lambda name: None)
    assert builder.build_binding() is None
    assert not old.exists() and "not built" in capsys.readouterr().out
    assert fl._lib._load_binding(fl._lib.lib(), old) is None
