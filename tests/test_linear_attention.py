"""``linear_attention`` on the CPU: the eager body against its recurrence in float64, its
gradients against differences, one token at a time, and its refusals."""

import math

import pytest
import torch

from mingru_amd import linear_attention, linear_attention_step


def recurrence(q, k, v, g, h=None, lengths=None, scale=None):
    """The definition, token by token, in the inputs' type."""
    B, T, Hk, dk = q.shape
    H, dv = v.shape[2:]
    scale = dk**-0.5 if scale is None else scale
    q, k = (t.repeat_interleave(H // Hk, 2) for t in (q, k))
    a = g.exp()
    a = torch.where(a < torch.finfo(torch.float32).tiny, 0 * a.detach(), a).expand(B, T, H)
    S = q.new_zeros(B, H, dk, dv) if h is None else h
    out = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool) if lengths is None else t < lengths
        live = live[:, None, None]
        kt, vt, qt = (torch.where(live, x[:, t], torch.zeros_like(x[:, t])) for x in (k, v, q))
        at = torch.where(live[..., 0], a[:, t], torch.ones_like(a[:, t]))
        S = at[..., None, None] * S + kt[..., None] * vt[..., None, :]
        out.append(scale * (qt[..., None] * S).sum(-2))
    return torch.stack(out, 1), S


def inputs(B, T, H, Hk, dk, dv, seed=0, documents=True, constant=False):
    r = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=r, dtype=torch.float64)  # noqa: E731
    q, k, v, h = n(B, T, Hk, dk), n(B, T, Hk, dk), n(B, T, H, dv), n(B, H, dk, dv)
    rate = torch.logspace(-2.5, 0, H, dtype=torch.float64)
    if constant:
        return q, k, v, -rate, h
    g = -rate * (0.1 + torch.rand(B, T, H, generator=r, dtype=torch.float64))
    if documents and T > 4:
        g[0, T // 2] = -math.inf
        g[-1, T // 3] = -1e30
        g[-1, T // 4] = -200.0
    return q, k, v, g, h


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 130])
@pytest.mark.parametrize("constant", [False, True])
def test_eager_matches_the_recurrence(T, constant):
    q, k, v, g, h = inputs(3, T, 4, 2, 5, 3, seed=T, constant=constant)
    lengths = torch.tensor([T, 0, min(T, 1)])
    for n in (None, lengths, lengths.int()):
        for h0 in (None, h):
            o, S = linear_attention(q, k, v, g, h0, n)
            wo, wS = recurrence(q, k, v, g, h0, n)
            assert torch.allclose(o, wo, rtol=1e-10, atol=1e-10)
            assert torch.allclose(S, wS, rtol=1e-10, atol=1e-10)


def test_gradients_match_differences():
    ts = [t.requires_grad_() for t in inputs(2, 70, 2, 1, 2, 3, documents=False)]
    lengths = torch.tensor([70, 66])
    assert torch.autograd.gradcheck(lambda *a: linear_attention(*a, lengths), ts, fast_mode=True)


def test_padding_is_not_read():
    q, k, v, g, h = inputs(2, 9, 2, 1, 4, 3, documents=False)
    lengths = torch.tensor([9, 4])
    want = linear_attention(q, k, v, g, h, lengths)
    for t in (q, k, v, g):
        t[1, 4:] = math.nan
    got = linear_attention(q, k, v, g, h, lengths)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert bool((got[0][1, 4:] == 0).all())


def test_steps_are_the_pass():
    q, k, v, g, h = inputs(2, 11, 4, 2, 5, 3)
    o, S = linear_attention(q, k, v, g, h, scale=0.3)
    for t in range(11):
        ot, h = linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], h, scale=0.3)
        assert torch.allclose(ot, o[:, t], rtol=1e-10, atol=1e-10)
    assert torch.allclose(h, S, rtol=1e-10, atol=1e-10)
    ot, h = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[0, 0])
    wo, wh = recurrence(q[:, :1], k[:, :1], v[:, :1], g[0, 0])
    assert torch.allclose(ot, wo[:, 0]) and torch.allclose(h, wh)


def test_no_tokens():
    q, k, v, g, h = inputs(2, 3, 2, 1, 4, 5)
    o, S = linear_attention(q[:, :0], k[:, :0], v[:, :0], g[:, :0], h)
    assert o.shape == (2, 0, 2, 5) and torch.equal(S, h)
    o, S = linear_attention(q[:0], k[:0], v[:0], g[:0])
    assert o.shape == (0, 3, 2, 5) and S.shape == (0, 2, 4, 5)


def test_types():
    q, k, v, g, h = (t.float() for t in inputs(2, 6, 2, 1, 4, 5))
    o, S = linear_attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), g, h)
    assert o.dtype == torch.bfloat16 and S.dtype == torch.float32
    o, S = linear_attention(q.bfloat16(), k.bfloat16(), v, g.bfloat16())
    assert o.dtype == torch.float32 and S.dtype == torch.float32


def test_refusals():
    q, k, v, g, h = inputs(2, 6, 4, 2, 4, 5)
    L = torch.tensor([6, 6])
    for bad, kind in (
        ((q, k[:, :5], v, g), ValueError), ((q, k, v[:, :, :3], g[..., :3]), ValueError),
        ((q, k, v, g[:, :5]), ValueError), ((q, k, v, g[..., 0]), ValueError),
        ((q[0], k[0], v[0], g[0]), ValueError), ((q, k, v, g, h[..., :4]), ValueError),
        ((q, k, v, g, h, L[:1]), ValueError), ((q, k, v, g, h, L.double()), TypeError),
        ((q, k, v, g, h, [6, 6]), TypeError), ((q.long(), k, v, g), TypeError),
        ((q[..., :0], k[..., :0], v, g), ValueError), ((q, k, v, g.to("meta")), ValueError),
    ):
        with pytest.raises(kind, match="linear_attention"):
            linear_attention(*bad)
    with pytest.raises(ValueError, match="linear_attention_step"):
        linear_attention_step(q, k, v, g)
