"""The build script's own behaviour: nothing is compiled here."""
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
