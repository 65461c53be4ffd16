"""The build script's own behaviour: nothing is compiled here."""
import sys

import pytest

import build_native


def test_force_ends_with_its_call(monkeypatch):
    seen = []
    monkeypatch.setattr(build_native, "ALL", {
        "one": lambda: seen.append(build_native.FORCE),
        "two": lambda: 1 / 0})
    build_native.build_all("one", force=True)
    assert seen == [True] and not build_native.FORCE
    with pytest.raises(ZeroDivisionError):
        build_native.build_all("two", force=True)
    assert not build_native.FORCE
    build_native.build_all("one")
    assert seen == [True, False]


def test_without_torch_the_binding_is_left_out(monkeypatch, capsys):
    """Everything else needs compilers only, and is built without it."""

    monkeypatch.setitem(sys.modules, "torch", None)
    monkeypatch.setattr(build_native, "_run", lambda cmd: pytest.fail(str(cmd)))
    assert build_native.build_paged_binding() is None
    assert "torch" in capsys.readouterr().out
