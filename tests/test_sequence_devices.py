"""``MINGRU_SCAN=hip`` with CPU tensors: the sequence operators decline, as the scans do, before any
native call sees a host pointer (CPU, the native calls stubbed)."""

import pytest

from mingru_amd import hip_scans, hip_sequence
from tests.test_sequence_forward_mode import CASES


@pytest.mark.parametrize("name", CASES)
def test_host_tensors_are_declined(monkeypatch, name):
    f, inputs = CASES[name]
    calls = []
    monkeypatch.setattr(hip_scans, "available", lambda: True)
    for stub in ("_stream", "_size"):
        monkeypatch.setattr(hip_sequence, stub, lambda *a: 256)
    monkeypatch.setattr(hip_sequence, "_call", lambda *a: calls.append(a[0]))
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    with pytest.raises(RuntimeError, match="need GPU tensors"):
        f(*inputs)
    with pytest.raises(RuntimeError, match="need GPU tensors"):
        f(*(t.clone().requires_grad_() for t in inputs))
    assert not calls
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    f(*inputs)
    assert not calls
