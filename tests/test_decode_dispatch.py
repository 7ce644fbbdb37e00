"""The decode operators follow ``MINGRU_SCAN``: CPU tensors under the forcing mode decline before any
native call, ``auto`` warns once and runs the eager body, and tangents leave the kernels."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mingru_amd import (
    beam_select,
    hip_scans,
    paged_attention_step,
    paged_cache_append,
    reorder_states,
    sequence_ops,
)

from tests.test_paged_cache import append_inputs, attend_inputs


def cases(dtype=torch.float32):
    s = append_inputs(2, 3, 2, 1, 4, 4, 2, 3, 2, dtype=dtype)
    a = attend_inputs(2, 4, 2, 8, 6, 4, 3, dtype=dtype)
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(2, 3, 7, generator=g).to(dtype)
    return {
        "paged_cache_append": (lambda q: paged_cache_append(**{**s, "q": q}), s["q"]),
        "paged_attention_step": (lambda q: paged_attention_step(**{**a, "q": q}), a["q"]),
        "beam_select": (lambda x: beam_select(x, torch.zeros(2, 3))[0], logits),
        "reorder_states": (lambda x: reorder_states(x, torch.tensor([[1, 0], [2, 2]])),
                           torch.randn(6, 5, generator=g)),
    }


NAMES = list(cases())


@pytest.mark.parametrize("name", NAMES)
def test_forcing_mode_on_the_cpu(monkeypatch, name):
    from mingru_amd import hip_decode

    f, x = cases()[name]
    calls = []
    monkeypatch.setattr(hip_decode, "_call", lambda *a: calls.append(a))
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    with pytest.raises(RuntimeError, match=name):
        f(x)
    assert not calls
    monkeypatch.setenv("MINGRU_SCAN", "nonsense")
    with pytest.raises(ValueError, match="MINGRU_SCAN"):
        f(x)


@pytest.mark.parametrize("name", NAMES)
def test_declines_warn_once(monkeypatch, name):
    from mingru_amd import hip_decode

    f, x = cases()[name]
    monkeypatch.setenv("MINGRU_SCAN", "eager")
    want = f(x)
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    monkeypatch.setattr(sequence_ops, "_warned", set())
    monkeypatch.setattr(hip_scans, "available", lambda: True)
    real = sequence_ops._dispatch
    from mingru_amd import decode_ops
    monkeypatch.setattr(decode_ops, "_dispatch", lambda what, is_cuda, *rest: real(what, True, *rest))

    def declines(*a):
        raise hip_scans.ScanFallback("not today")

    monkeypatch.setattr(hip_decode, f"{name}_impl", declines)
    with pytest.warns(UserWarning, match="not today"):
        assert torch.equal(f(x), want)
    import warnings
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert torch.equal(f(x), want)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_leave_the_kernels(monkeypatch, name):
    from mingru_amd import decode_ops, hip_decode

    f, x = cases()[name]
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    monkeypatch.setattr(sequence_ops, "_warned", set())
    monkeypatch.setattr(hip_scans, "available", lambda: True)
    real = sequence_ops._dispatch
    monkeypatch.setattr(decode_ops, "_dispatch", lambda what, is_cuda, *rest: real(what, True, *rest))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)  # the CPU's index
    monkeypatch.setattr(hip_decode, "_stream", lambda t: 0)
    monkeypatch.setattr(hip_decode, "_size", lambda *a: 256)
    calls = []
    monkeypatch.setattr(hip_decode, "_call", lambda *a: calls.append(a[0]))
    f(x)
    assert len(calls) == 1
    with forward_ad.dual_level():
        with pytest.warns(UserWarning, match="forward-mode"):
            out = f(forward_ad.make_dual(x, torch.ones_like(x)))
        assert forward_ad.unpack_dual(out).tangent is not None
    assert len(calls) == 1


def test_calls_run_on_their_tensors_device(monkeypatch):
    """The default stream is a number that means the current device's."""
    import contextlib

    from mingru_amd import hip_decode

    class Tensor:
        device = torch.device("cuda", 1)

    current = [0]

    @contextlib.contextmanager
    def device(d):
        old, current[0] = current[0], d.index
        yield
        current[0] = old

    seen = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(hip_decode, "_stream", lambda t: 0)
    monkeypatch.setattr(hip_decode, "_call", lambda *a: seen.append((current[0], a)))
    hip_decode._launch("what", Tensor(), "name", 3)
    current[0] = 1
    hip_decode._launch("what", Tensor(), "name", 3)
    assert seen == [(1, ("name", 3, 0))] * 2 and current == [1]
