"""``linear_cross_entropy`` on the CPU: the eager body against the definition in float64, its
gradients against differences and the formulas, and its refusals."""

import math

import pytest
import torch

from mingru_amd import linear_cross_entropy


def inputs(N, V, D, seed=0, ignored=0.3, bias=True):
    r = torch.Generator().manual_seed(seed)
    x = torch.randn(N, D, generator=r, dtype=torch.float64)
    w = torch.randn(V, D, generator=r, dtype=torch.float64) * (1.5 / math.sqrt(D))
    b = torch.randn(V, generator=r, dtype=torch.float64) * 0.5 if bias else None
    t = torch.randint(0, V, (N,), generator=r)
    t[torch.rand(N, generator=r) < ignored] = -100
    return x, w, t, b


def plain(x, w, t, b, reduction="mean", up=None):
    """Loss and gradients from the formulas, row by row's softmax written out."""
    keep = t != -100
    l = x @ w.t() + (0 if b is None else b)
    top = l.max(-1, keepdim=True).values
    e = (l - top).exp()
    p = e / e.sum(-1, keepdim=True)
    at = torch.where(keep, t, torch.zeros_like(t))
    each = (e.sum(-1).log() + top[:, 0] - l.gather(1, at[:, None])[:, 0]) * keep
    n = max(1, int(keep.sum()))
    up = torch.ones(()) if up is None else up
    g = {"none": up, "sum": up, "mean": up / n}[reduction] * keep
    d = p * g[:, None]
    d.scatter_add_(1, at[:, None], -g[:, None].to(d.dtype))
    loss = {"none": each, "sum": each.sum(), "mean": each.sum() / n}[reduction]
    return loss, d @ w, d.t() @ x, d.sum(0)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("bias", [True, False])
def test_eager_matches_the_definition(reduction, bias):
    x, w, t, b = inputs(7, 11, 5, bias=bias)
    ts = [v.requires_grad_() for v in (x, w, b) if v is not None]
    loss = linear_cross_entropy(x, w, t, b, reduction=reduction)
    up = torch.randn(loss.shape, dtype=torch.float64)
    got = torch.autograd.grad(loss, ts, up)
    with torch.no_grad():
        want = plain(x, w, t, b, reduction, up)
    assert torch.allclose(loss, want[0], rtol=1e-12)
    for a, c in zip(got, want[1:]):
        assert torch.allclose(a, c, rtol=1e-10, atol=1e-12)


def test_gradients_match_differences():
    x, w, t, b = inputs(4, 5, 3)
    ts = [v.requires_grad_() for v in (x, w, b)]
    assert torch.autograd.gradcheck(lambda x, w, b: linear_cross_entropy(x, w, t, b), ts)


def test_nothing_counts():
    x, w, t, b = inputs(4, 5, 3)
    t[:] = -100
    x[1] = math.nan
    for v in (x, w, b):
        v.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(x, w, t, b, reduction=reduction)
        assert bool((loss == 0).all())
        for g in torch.autograd.grad(loss.sum(), (x, w, b)):
            assert bool((g == 0).all())
    x, w, t, b = inputs(0, 5, 3)
    assert linear_cross_entropy(x, w, t, b).item() == 0
    assert linear_cross_entropy(x, w, t, b, reduction="none").shape == (0,)


def test_left_out_rows_are_not_read():
    x, w, t, b = inputs(6, 5, 3, ignored=0)
    t[2] = 4
    want = linear_cross_entropy(x[[0, 1, 3, 4, 5]], w, t[[0, 1, 3, 4, 5]], b)
    t[2], x[2] = 7, math.inf
    assert torch.equal(linear_cross_entropy(x, w, t, b, ignore_index=7), want)


def test_shapes_and_types():
    x, w, t, b = inputs(6, 5, 3)
    loss = linear_cross_entropy(x.view(2, 3, 3), w, t.view(2, 3), b, reduction="none")
    assert loss.shape == (2, 3)
    loss = linear_cross_entropy(x.bfloat16(), w.bfloat16(), t.int(), b.float())
    assert loss.dtype == torch.float32


def test_refusals():
    x, w, t, b = inputs(4, 5, 3)
    for args, kw, kind in (
        ((x, w[:, :2], t, b), {}, ValueError), ((x, w[0], t, b), {}, ValueError),
        ((x, w, t[:3], b), {}, ValueError), ((x, w, t, b[:4]), {}, ValueError),
        ((x, w, t.double(), b), {}, TypeError), ((x, w, [1, 2, 3, 4], b), {}, TypeError),
        ((x, w, t > 0, b), {}, TypeError), ((x.long(), w, t, b), {}, TypeError),
        ((x, w, t, b), dict(reduction="median"), ValueError),
        ((x, w[:0], t, b[:0]), {}, ValueError), ((x, w.to("meta"), t, b), {}, ValueError),
        ((x, w, torch.full((4,), 5), b), {}, IndexError),
        ((x, w, torch.full((4,), -1), b), {}, IndexError),
    ):
        with pytest.raises(kind, match="linear_cross_entropy"):
            linear_cross_entropy(*args, **kw)
