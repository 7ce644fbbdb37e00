"""``linear_cross_entropy`` with ``reduction="none"`` in fp32: rows' upstream gradients of any size leave
each row's own gradient as exact as it is alone, and left-out rows' have no effect.

Tolerances, of each row's norm: as for a whole tensor (test_gpu_linear_cross_entropy.py), 1e-5: a
row of ``dx`` is its upstream gradient times what the other rows do not enter.  ``dw`` and ``db`` sum
over rows, so theirs is of the whole tensor's norm."""

import math

import pytest
import torch

from mingru_amd import linear_cross_entropy
from tests.test_linear_cross_entropy import inputs, plain

pytestmark = pytest.mark.gpu

TOL = 1e-5


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


def check(cuda, N, up_of, scale=1.0, bias=True):
    x, w, t, b = inputs(N, 700, 96, seed=N, bias=bias)
    r = torch.Generator().manual_seed(1)
    up = up_of(torch.randn(N, generator=r, dtype=torch.float64), t == -100).float()
    x, w, b = (None if v is None else v.float() for v in (x, w, b))
    counted = up.double().masked_fill(t == -100, 0)  # plain multiplies, and 0 times a NaN is one
    want = plain(x.double(), w.double(), t, None if b is None else b.double(), "none", counted)
    ts = [v.to(cuda).requires_grad_() for v in (x, w, b) if v is not None]
    loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2] if bias else None, reduction="none")
    grads = torch.autograd.grad(loss, ts, up.to(cuda))
    dx, wdx = grads[0].double().cpu(), want[1]
    rows = (dx - wdx).norm(dim=1) / wdx.norm(dim=1).clamp(min=1e-300)
    errors = [off(a, c) for a, c in zip(grads, want[1:])]
    print("rows", float(rows.max()), "dx dw db", errors, flush=True)
    assert bool((dx[t == -100] == 0).all())
    assert float(rows.max()) <= TOL and max(errors) <= TOL


@pytest.mark.parametrize("N", [100, 200, 700])
@pytest.mark.parametrize("bias", [True, False])
def test_left_out_rows_have_no_effect(cuda, N, bias):
    check(cuda, N, lambda u, out: torch.where(out, torch.full_like(u, 1e12), u), bias=bias)
    check(cuda, N, lambda u, out: torch.where(out, torch.full_like(u, math.nan), u), bias=bias)


@pytest.mark.parametrize("N", [100, 200, 700])
@pytest.mark.parametrize("lowest", [-6, -12, -25])
def test_weights_of_many_sizes(cuda, N, lowest):
    check(cuda, N, lambda u, out: u * torch.logspace(0, lowest, len(u), dtype=u.dtype))


@pytest.mark.parametrize("N", [100, 200])
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e20])
def test_weights_of_one_size(cuda, N, size):
    check(cuda, N, lambda u, out: u * size)


def test_a_weight_that_is_not_finite_stays_in_its_row(cuda):
    x, w, t, b = (v.to(cuda) for v in inputs(200, 300, 64, ignored=0.0))
    x, w, b = (v.float().requires_grad_() for v in (x, w, b))
    loss = linear_cross_entropy(x, w, t, b, reduction="none")
    up = torch.ones(200, device=cuda)
    want, = torch.autograd.grad(loss, x, up, retain_graph=True)
    up[7] = math.inf
    got, = torch.autograd.grad(loss, x, up)
    assert not bool(got[7].isfinite().any())
    keep = torch.arange(200, device=cuda) != 7
    assert torch.equal(got[keep], want[keep])
