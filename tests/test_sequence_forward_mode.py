"""Forward-mode derivatives of the sequence operators: calls with a tangent leave the kernels, which
have none, to the eager bodies (CPU, the native calls stubbed; and on the GPU)."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mingru_amd import (
    hip_scans,
    linear_attention,
    linear_attention_step,
    linear_cross_entropy,
    residual_norm,
    sequence_ops,
)


def _cases():
    r = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=r)  # noqa: E731
    target = torch.tensor([1, 4, -100])
    return {
        "residual_norm": (lambda h, x, g, w: residual_norm(h, x, gate=g, pre_weight=w),
                          [n(3, 8), n(3, 8), n(3, 8), n(8)]),
        "linear_attention": (linear_attention,
                             [n(2, 5, 1, 4), n(2, 5, 1, 4), n(2, 5, 2, 3), -n(2, 5, 2).abs(),
                              n(2, 2, 4, 3)]),
        "linear_attention_step": (linear_attention_step,
                                  [n(2, 1, 4), n(2, 1, 4), n(2, 2, 3), -n(2, 2).abs(),
                                   n(2, 2, 4, 3)]),
        "linear_cross_entropy": (lambda x, w, b: linear_cross_entropy(x, w, target.to(x.device), b),
                                 [n(3, 4), n(5, 4), n(5)]),
    }


CASES = _cases()


def _tangents(f, inputs, which):
    """The outputs' tangents with a tangent of ones on input ``which``."""
    with forward_ad.dual_level():
        inputs = list(inputs)
        inputs[which] = forward_ad.make_dual(inputs[which], torch.ones_like(inputs[which]))
        out = f(*inputs)
        out = out if isinstance(out, tuple) else (out,)
        return [forward_ad.unpack_dual(t).tangent for t in out]


WHICH = [(name, i) for name, (_, inputs) in CASES.items() for i in range(len(inputs))]


@pytest.mark.parametrize("name, which", WHICH)
def test_tangents_are_not_dropped(monkeypatch, name, which):
    from mingru_amd import hip_sequence

    f, inputs = CASES[name]
    want = _tangents(f, inputs, which)
    calls = []
    dispatch = sequence_ops._dispatch  # as on the GPU
    monkeypatch.setattr(sequence_ops, "_dispatch", lambda what, is_cuda, call: dispatch(what, True, call))
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    monkeypatch.setattr(sequence_ops, "_warned", set())
    monkeypatch.setattr(hip_scans, "available", lambda: True)
    monkeypatch.setattr(hip_sequence, "_stream", lambda t: 0)
    monkeypatch.setattr(hip_sequence, "_size", lambda *a: 256)
    monkeypatch.setattr(hip_sequence, "_call", lambda *a: calls.append(a[0]))
    f(*inputs)
    assert len(calls) == 1  # without a tangent the kernels run, inside of a level too
    with forward_ad.dual_level():
        f(*inputs)
    assert len(calls) == 2
    with pytest.warns(UserWarning, match="forward-mode"):
        got = _tangents(f, inputs, which)
    assert len(calls) == 2
    assert all(torch.equal(a, b) for a, b in zip(got, want) if b is not None)
    assert [t is None for t in got] == [t is None for t in want]


@pytest.mark.gpu
@pytest.mark.parametrize("name, which", WHICH)
def test_tangents_on_the_gpu(cuda, monkeypatch, name, which):
    f, inputs = CASES[name]
    dev = [t.to(cuda) for t in inputs]
    want = _tangents(f, [t.double() for t in inputs], which)
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    monkeypatch.setattr(sequence_ops, "_warned", set())
    with pytest.warns(UserWarning, match="forward-mode"):
        got = _tangents(f, dev, which)
    for a, b in zip(got, want):
        # Sums of at most 16 terms in 32 bits, a few in a row.
        assert (a is None) == (b is None)
        assert b is None or float((a.double().cpu() - b).norm()) <= 64 * 2.0**-24 * max(1.0, float(b.norm()))
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    with pytest.raises(RuntimeError, match="forward-mode"):
        _tangents(f, dev, which)
