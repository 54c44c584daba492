"""CPU: which libraries the binding takes."""
import pytest

from flash_tree_attn_b200 import _lib


class _Library:
    """Exports `names`; reports `version`."""

    def __init__(self, names, version):
        for name in names:
            setattr(self, name, type("entry", (), {"__call__": staticmethod(lambda *a: version)})())


@pytest.mark.parametrize("gone", [["fta_token_logprobs"], ["fta_decode_token", "fta_evict_rows"]])
def test_a_library_that_lacks_an_entry_is_refused_by_name(monkeypatch, fta_lib, gone):
    """An older build of the same ABI version, as FTA_LIB_PATH may name it."""
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.C, "CDLL", lambda path: _Library([n for n in _lib.SYMBOLS if n not in gone], _lib.ABI_VERSION))
    with pytest.raises(_lib.FtaLibraryMissing, match="lacks " + ", ".join(gone) + ": rebuild"):
        _lib.load()
    assert _lib._lib is None


def test_another_version_is_refused_and_a_whole_library_taken(monkeypatch, fta_lib):
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.C, "CDLL", lambda path: _Library(_lib.SYMBOLS, 100))
    with pytest.raises(_lib.FtaLibraryMissing, match="ABI version 100"):
        _lib.load()
    whole = _Library(_lib.SYMBOLS, _lib.ABI_VERSION)
    monkeypatch.setattr(_lib.C, "CDLL", lambda path: whole)
    assert _lib.load() is whole
