"""``residual_norm`` on the CPU: the eager body against the formulas in float64, its
gradients against differences, and its refusals."""

import pytest
import torch

from mingru_amd import residual_norm


def plain(h, x, post, post_w, post_b, gate, act, scale, pre, pre_w, pre_b, eps=1e-5):
    """The definition, element by element of numpy-like float64 tensors."""
    def norm(v, kind, w, b):
        if kind == "layer":
            mean = v.sum(-1, keepdim=True) / v.shape[-1]
            var = ((v - mean) ** 2).sum(-1, keepdim=True) / v.shape[-1]
            v = (v - mean) / (var + eps) ** 0.5
        elif kind == "rms":
            v = v / ((v * v).sum(-1, keepdim=True) / v.shape[-1] + eps) ** 0.5
        v = v if w is None else v * w
        return v if b is None else v + b

    u = norm(h, post, post_w, post_b) if post != "none" else h
    if gate is not None:
        s = 1 / (1 + (-gate).exp())
        u = u * (s * gate if act == "silu" else s)
    r = u if x is None else x + (u if scale is None else scale * u)
    return (r,) if pre == "none" else (r, norm(r, pre, pre_w, pre_b))


def inputs(shape, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    big = [torch.randn(*shape, generator=g, dtype=torch.float64) for _ in range(3)]
    vec = [1 + 0.3 * torch.randn(D, generator=g, dtype=torch.float64) for _ in range(5)]
    return [t.to(dtype) for t in big + vec]


@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("act", [None, "sigmoid", "silu"])
@pytest.mark.parametrize("pre", ["none", "layer", "rms"])
def test_eager_matches_the_definition(post, act, pre):
    h, x, gate, scale, pw, pb, qw, qb = inputs((2, 3, 7))
    gate = None if act is None else gate
    pw, pb = (None, None) if post == "none" else (pw, pb)
    qw, qb = (None, None) if pre == "none" else (qw, qb)
    got = residual_norm(h, x, post=post, post_weight=pw, post_bias=pb, gate=gate,
                        gate_act=act or "silu", scale=scale, pre=pre, pre_weight=qw, pre_bias=qb)
    got = got if isinstance(got, tuple) else (got,)
    want = plain(h, x, post, pw, pb, gate, act, scale, pre, qw, qb)
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_gradients_match_differences():
    ts = [t.requires_grad_() for t in inputs((2, 5))]
    assert torch.autograd.gradcheck(
        lambda h, x, g, s, pw, pb, qw, qb: residual_norm(
            h, x, post="layer", post_weight=pw, post_bias=pb, gate=g, gate_act="silu", scale=s,
            pre="rms", pre_weight=qw, pre_bias=qb), ts)


def test_number_scale_and_broadcast_gate():
    h, x, gate = inputs((2, 3, 4))[:3]
    r = residual_norm(h, x, gate=gate[:, :1], gate_act="sigmoid", scale=0.25, pre="none")
    assert torch.allclose(r, x + 0.25 * h * torch.sigmoid(gate[:, :1]))
    assert residual_norm(h.bfloat16(), x.float(), pre="none").dtype == torch.float32


def test_refusals():
    h, x, gate, scale, w = inputs((2, 4))[:5]
    for bad, kind in (
        (dict(x=x[:, :2]), ValueError), (dict(post="batch"), ValueError),
        (dict(pre=None), ValueError), (dict(gate=gate, gate_act="relu"), ValueError),
        (dict(scale=scale), ValueError), (dict(scale=2.0), ValueError),
        (dict(x=x, scale=scale[:2]), ValueError), (dict(post_weight=w), ValueError),
        (dict(pre="none", pre_bias=w), ValueError), (dict(pre_weight=w[:3]), ValueError),
        (dict(x=x.long()), TypeError), (dict(gate=1.0), TypeError),
        (dict(x=x.to("meta")), ValueError),
    ):
        with pytest.raises(kind, match="residual_norm"):
            residual_norm(h, **bad)
    with pytest.raises(ValueError, match="last dimension"):
        residual_norm(torch.tensor(1.0))
    with pytest.raises(RuntimeError):
        residual_norm(h, gate=gate[:, :3])  # does not broadcast


def test_empty_rows():
    h = torch.zeros(0, 8)
    r, y = residual_norm(h, h)
    assert r.shape == y.shape == (0, 8)
