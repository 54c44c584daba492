"""CPU: how the decoding-loop entries call the C library (current device, stream, error codes), with fakes."""
import pytest
import torch

from flash_tree_attn_b200 import _lib


class _Device:
    current = 0

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.before, _Device.current = _Device.current, self.index

    def __exit__(self, *exc):
        _Device.current = self.before


@pytest.mark.parametrize("index", [0, 3])
def test_the_tensors_device_is_current_during_the_call(monkeypatch, index):
    _Device.current = 0
    monkeypatch.setattr(_lib, "_current_device", lambda: _Device.current)
    monkeypatch.setattr(_lib, "_raw_stream", lambda i: 1000 + i)
    monkeypatch.setattr(torch.cuda, "device", _Device)
    seen = []

    def entry(p, stream):
        seen.append((p, stream, _Device.current))
        return _lib.FTA_OK

    _lib.launch(entry, b"parameters", index, "entry")
    assert seen == [(b"parameters", 1000 + index, index)] and _Device.current == 0


def test_an_error_code_becomes_an_exception_and_the_device_comes_back(monkeypatch, fta_lib):
    _Device.current = 0
    monkeypatch.setattr(_lib, "_current_device", lambda: _Device.current)
    monkeypatch.setattr(_lib, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(torch.cuda, "device", _Device)
    with pytest.raises(_lib.FtaError) as e:
        _lib.launch(lambda p, s: _lib.FTA_E_BADARG, b"", 2, "entry")
    assert e.value.code == _lib.FTA_E_BADARG and "entry" in str(e.value) and _Device.current == 0


@pytest.mark.parametrize("cls,pack", [(_lib.FtaTokenParams, _lib.pack_token), (_lib.FtaRotaryParams, _lib.pack_rotary),
                                      (_lib.FtaEvictParams, _lib.pack_evict), (_lib.FtaLogprobParams, _lib.pack_logprob)])
def test_packed_parameters_are_the_structure(cls, pack):
    """Every field's own value, packed in one step, lands where the ctypes mirror has it."""
    values = [0.5 if t is _lib._f32 else i + 1 for i, (_, t) in enumerate(cls._fields_)]
    p = cls.from_buffer_copy(pack(*values))
    assert [getattr(p, name) for name, _ in cls._fields_] == values


def test_rows_of():
    t = torch.zeros(2, 3, 4, 64, dtype=torch.float16)
    assert _lib.rows_of(t) == (t.data_ptr(), 768, 256, 64)
    assert _lib.rows_of(t[..., 1:33]) is None          # an odd address
    assert _lib.rows_of(t[..., ::2]) is None           # elements apart
    assert _lib.rows_of(t[..., :60].clone()) is None   # rows of 120 bytes
