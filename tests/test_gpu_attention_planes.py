"""fp32 outputs of bf16 inputs carry the bits of three bf16 planes: the states, and the decays'
gradient, whose operands (decayed rows, the state) are split into them.

Tolerances, as the 2-norm of the difference over the 2-norm of the result.  A value in three planes is
exact to 2^-27, in two to 2^-18.  What is left with three are the sums' roundings, 2^-25 rms each: a
state of decay a token keeps the last few hundred tokens, 6 sums for each 64 of them, and the
weights' exponentials, 2^-24: 2^-25 * sqrt(6 * 16 + 4) = 3e-7; 1e-6 allows for three times that.
The decays' gradient sums terms that cancel: twice the states' bound.  With two planes the operands'
roundings alone exceed both (test_two_planes_would_not_do)."""

import math

import pytest
import torch

from mingru_amd import linear_attention
from tests.test_linear_attention import inputs, recurrence

STATE, DECAY = 1e-6, 2e-6


def off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


@pytest.mark.gpu
@pytest.mark.parametrize("B, T, H, Hk", [(1, 700, 2, 2), (2, 1000, 4, 2), (4, 200, 64, 64)])
@pytest.mark.parametrize("documents", [False, True])
def test_states_and_decays(cuda, monkeypatch, B, T, H, Hk, documents):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    d = 128
    vals = inputs(B, T, H, Hk, d, d, seed=T, documents=documents)
    vals = [t.bfloat16() for t in vals[:3]] + [t.float() for t in vals[3:]]
    r = torch.Generator().manual_seed(5)
    do = torch.randn(B, T, H, d, generator=r).bfloat16()
    dh = torch.randn(B, H, d, d, generator=r)
    ref = [t.to(cuda).double().requires_grad_() for t in vals]
    want = on_device(*ref)
    wgrads = torch.autograd.grad(want, ref[3:], (do.to(cuda).double(), dh.to(cuda).double()))
    dev = [t.to(cuda).requires_grad_() for t in vals]
    got = linear_attention(*dev)
    grads = torch.autograd.grad(got, dev[3:], (do.to(cuda), dh.to(cuda)))
    errors = {"h": off(got[1], want[1]) / STATE, "dg": off(grads[0], wgrads[0]) / DECAY,
              "dh0": off(grads[1], wgrads[1]) / STATE}
    print({n: round(e, 3) for n, e in errors.items()}, flush=True)
    assert max(errors.values()) <= 1, errors


def on_device(q, k, v, g, h):
    """The recurrence in chunks of 50 tokens, as products in float64 on the inputs' device."""
    B, T, Hk, dk = q.shape
    H = v.shape[2]
    q, k = (t.repeat_interleave(H // Hk, 2).transpose(1, 2) for t in (q, k))
    v, g = v.transpose(1, 2), g.transpose(1, 2)
    out = []
    for at in range(0, T, 50):
        qc, kc, vc, gc = (t[:, :, at : at + 50] for t in (q, k, v, g))
        n = gc.shape[-1]
        start = gc < math.log(torch.finfo(torch.float32).tiny)
        G = torch.where(start, torch.zeros_like(gc), gc).cumsum(-1)
        count = start.cumsum(-1)
        seen = (count[..., :, None] == count[..., None, :]) & torch.ones(
            n, n, dtype=torch.bool, device=q.device).tril()
        D = torch.where(seen, (G[..., :, None] - G[..., None, :]).masked_fill(~seen, 0).exp(), 0.0)
        c = torch.where(count == 0, G.exp(), 0.0)
        o = c[..., None] * (qc @ h) + ((qc @ kc.transpose(-1, -2).contiguous()) * D) @ vc
        out.append(dk**-0.5 * o)
        h = c[..., -1, None, None] * h + (kc * D[..., -1, :, None]).transpose(-1, -2).contiguous() @ vc
    return torch.cat(out, 2).transpose(1, 2), h


def test_the_chunked_reference():
    q, k, v, g, h = inputs(2, 120, 4, 2, 8, 6)
    for a, b in zip(on_device(q, k, v, g, h), recurrence(q, k, v, g, h)):
        assert off(a, b) <= 1e-13


def _planes(x, n):
    """What ``n`` planes of 8 bits hold of ``x``."""
    held = torch.zeros_like(x)
    for _ in range(n):
        held = held + (x - held).float().bfloat16().double()
    return held


def _state_and_decays(q, k, v, g, h, do, dh, held):
    """The final state and the decays' gradient, chunk by chunk in float64 but for what ``held``
    makes of the operands that the states are built from and of the states as operands."""
    T = q.shape[2]
    G = g.cumsum(-1)
    chunks = [slice(at, at + 64) for at in range(0, T, 64)]
    base = lambda c: G[..., c.start - 1 : c.start] if c.start else torch.zeros_like(G[..., :1])  # noqa: E731
    e = torch.zeros_like(G)

    def inner(c):
        """Pairs of a chunk: ``X_ij``, which both sides take."""
        n = G[..., c].shape[-1]
        lower = torch.ones(n, n, dtype=torch.bool).tril(-1)
        D = torch.where(lower, (G[..., c][..., :, None] - G[..., c][..., None, :]).exp(), 0.0)
        return D * (q[:, :, c] @ k[:, :, c].transpose(-1, -2)) * (do[:, :, c] @ v[:, :, c].transpose(-1, -2))

    S = h
    for c in chunks:
        dq = (G[..., c] - base(c)).exp()[..., None] * (do[:, :, c] @ held(S).transpose(-1, -2))
        X = inner(c)
        e[..., c] = (q[:, :, c] * dq).sum(-1) + X.sum(-1) - X.sum(-2)
        w = (G[..., c][..., -1:] - G[..., c]).exp()
        keep = (G[..., c][..., -1] - base(c)[..., 0]).exp()
        S = keep[..., None, None] * S + held(k[:, :, c] * w[..., None]).transpose(-1, -2) @ v[:, :, c]
    R = dh
    for c in reversed(chunks):
        w = (G[..., c][..., -1:] - G[..., c]).exp()
        dk = w[..., None] * (v[:, :, c] @ held(R).transpose(-1, -2))
        e[..., c] -= (k[:, :, c] * dk).sum(-1)
        up = (G[..., c] - base(c)).exp()[..., None]
        keep = (G[..., c][..., -1] - base(c)[..., 0]).exp()
        R = keep[..., None, None] * R + held(q[:, :, c] * up).transpose(-1, -2) @ do[:, :, c]
    return S, e.flip(-1).cumsum(-1).flip(-1) + (S * dh).sum((-1, -2))[..., None]


def test_two_planes_would_not_do():
    """The operands' roundings in float64 sums otherwise: two planes exceed the bounds above, three
    are far within."""
    T, d, H = 700, 128, 2
    vals = inputs(1, T, H, H, d, d, seed=T, documents=False)
    vals = [t.bfloat16().double() for t in vals[:3]] + list(vals[3:])
    r = torch.Generator().manual_seed(5)
    do = torch.randn(1, T, H, d, generator=r).bfloat16().double()
    dh = torch.randn(1, H, d, d, generator=r, dtype=torch.float64)
    ref = [t.clone().requires_grad_() for t in vals]
    want = on_device(*ref)
    dg = torch.autograd.grad(want, ref[3], (do * d**0.5, dh))[0]
    q, k, v, g, do = (t.transpose(1, 2) for t in (*vals[:4], do))
    for n, held in ((None, lambda x: x), (2, lambda x: _planes(x, 2)), (3, lambda x: _planes(x, 3))):
        S, e = _state_and_decays(q, k, v, g, vals[4], do, dh, held)
        errors = off(S, want[1]), off(e, dg.transpose(1, 2))
        print(n, errors)
        if n is None:
            assert max(errors) <= 1e-12
        elif n == 2:
            assert errors[0] > STATE and errors[1] > DECAY
        else:
            assert errors[0] < STATE / 20 and errors[1] < DECAY / 20
