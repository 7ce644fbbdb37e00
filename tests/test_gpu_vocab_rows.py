"""``linear_cross_entropy`` in fp32: a row's loss and gradient do not depend on how large other rows
are.  Tolerance, of each row's loss and gradient: 1e-5, as for a whole tensor of rows of one size
(test_gpu_linear_cross_entropy.py: logits' absolute error; theirs are of size 5 at most here but
in the large rows, which are compared by their own logits' size)."""

import pytest
import torch

from mingru_amd import linear_cross_entropy
from tests.test_linear_cross_entropy import inputs, plain

pytestmark = pytest.mark.gpu

TOL = 1e-5


@pytest.mark.parametrize("N", [100, 200, 600])
@pytest.mark.parametrize("large", [1e4, 1e8, 1e20])
def test_rows_of_many_sizes(cuda, monkeypatch, N, large):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    x, w, t, b = inputs(N, 700, 96, seed=N, ignored=0.1)
    t[5:9] = torch.arange(4)
    x[5:9] *= large
    x, w, b = (v.float() for v in (x, w, b))
    up = torch.ones(N)
    up[5:9] = 1 / large
    want = plain(x.double(), w.double(), t, b.double(), "none", up.double())
    ts = [v.to(cuda).requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2], reduction="none")
    grads = [g.double().cpu() for g in torch.autograd.grad(loss, ts, up.to(cuda))]
    loss = loss.detach().double().cpu()
    size = torch.ones(N, dtype=torch.float64)
    size[5:9] = large
    each = ((loss - want[0]).abs() / (size * want[0].abs().clamp(min=1.0)))
    small = torch.ones(N, dtype=torch.bool)
    small[5:9] = False  # a large row's softmax is a comparison: its gradient may turn on a rounding
    rows = ((grads[0] - want[1]).norm(dim=1) / want[1].norm(dim=1).clamp(min=1e-300))[small]
    errors = [float((a - c).norm() / c.norm()) for a, c in zip(grads[1:], want[2:])]
    print("loss", float(each.max()), "rows", float(rows.max()), "dw db", errors, flush=True)
    assert float(each.max()) <= TOL and float(rows.max()) <= TOL and max(errors) <= TOL


@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_small_rows_beside_a_large_one(cuda, monkeypatch, reduction):
    """The large row's loss is about 0: the sum is the small rows'."""
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    x, w, t, b = inputs(300, 700, 96, ignored=0.1)
    x[17] *= 1e8
    t[17] = (x[17] @ w.t()).argmax()
    x, w, b = (v.float() for v in (x, w, b))
    want = plain(x.double(), w.double(), t, b.double(), reduction)
    ts = [v.to(cuda).requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2], reduction=reduction)
    got = [v.detach().double().cpu() for v in (loss, *torch.autograd.grad(loss, ts))]
    errors = [float((a - c).norm() / c.norm()) for a, c in zip(got, want)]
    print(errors, flush=True)
    assert max(errors) <= TOL
