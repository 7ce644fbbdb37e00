"""``linear_cross_entropy`` kernels against the formulas in float64: rows, vocabularies and
widths around the tiles, left-out rows, pieces of the vocabulary, reductions, streams, graphs.

Tolerances, as the 2-norm of the difference over the 2-norm of the result.  Logits are sums of D
products in fp32, sqrt(D) 2^-24 of their terms' size each; the loss and the probabilities take
over their absolute error, with terms of size at most 5 here: for D up to 1100, 5 * 33 * 2^-24
= 1e-5.  The gradients' products sum V or N terms of either sign, sqrt(V) 2^-24: less.  fp32:
1e-5 (the probabilities' error is relative to them, so it carries over once).  bf16 gradients:
d and the result are rounded to 8 bits, 2 * 2^-8.
"""

import math

import pytest
import torch

from mingru_amd import linear_cross_entropy
from tests.test_linear_cross_entropy import inputs, plain

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2 * 2.0**-8, torch.float16: 1e-5 + 2.0**-11}


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


def check(cuda, N, V, D, dtype, reduction="mean", bias=True, ignored=0.3, seed=0,
          layout=lambda t: t):
    x, w, t, b = inputs(N, V, D, seed, ignored, bias)
    x, w, b = (None if v is None else v.to(dtype) for v in (x, w, b))
    r = torch.Generator().manual_seed(seed + 1)
    up = torch.randn((N,) if reduction == "none" else (), generator=r)
    want = plain(*(None if v is None else v.double() for v in (x, w)), t,
                 None if b is None else b.double(), reduction, up.double())
    dev = [layout(x.to(cuda)).requires_grad_(), w.to(cuda).requires_grad_(),
           None if b is None else b.to(cuda).requires_grad_()]
    loss = linear_cross_entropy(dev[0], dev[1], t.to(cuda), dev[2], reduction=reduction)
    grads = torch.autograd.grad(loss, [v for v in dev if v is not None], up.to(cuda))
    assert loss.dtype == torch.float32
    errors = {"loss": off(loss, want[0]) / 1e-5}
    for n, a, c, v in zip(("dx", "dw", "db"), grads, want[1:], dev):
        assert a.shape == v.shape and a.dtype == dtype
        errors[n] = off(a, c) / TOL[dtype] if float(c.norm()) else float(a.abs().max())
    print({n: round(e, 3) for n, e in errors.items()}, flush=True)
    assert max(errors.values()) <= 1, errors


@pytest.mark.parametrize("N, V, D", [(1, 1, 1), (1, 300, 64), (3, 5, 2), (63, 257, 65),
                                     (256, 256, 64), (257, 1000, 128), (300, 513, 100),
                                     (1000, 2000, 392), (65, 700, 1088)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(cuda, N, V, D, dtype):
    check(cuda, N, V, D, dtype, seed=N, ignored=0.0 if N < 4 else 0.3)


@pytest.mark.parametrize("N, V, D", [(1, 1, 4), (2, 31, 7), (31, 33, 5), (32, 129, 36), (33, 640, 31),
                                     (64, 1000, 129), (90, 100, 1001), (128, 5003, 66),
                                     (129, 130, 33), (8, 4099, 1000)])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_few_rows(cuda, N, V, D, reduction):
    """Up to 128 fp32 rows have kernels of their own; whole vectors of bf16 weights lie in place."""
    check(cuda, N, V, D, torch.float32, reduction, bias=V % 2 == 0, seed=N, ignored=0.2 if N > 8 else 0)
    check(cuda, N, V, D - D % 8 + 8, torch.bfloat16, reduction, seed=N)


def test_few_rows_left_out(cuda):
    for N in (20, 60, 120):
        check(cuda, N, 300, 64, torch.float32, "none", ignored=0.9)
        check(cuda, N, 300, 64, torch.float32, "none", ignored=1.0)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_reductions(cuda, reduction, bias, dtype):
    check(cuda, 130, 400, 192, dtype, reduction, bias)


@pytest.mark.parametrize("ignored", [0.0, 0.9, 1.0])
def test_left_out_rows(cuda, ignored):
    check(cuda, 600, 300, 64, torch.bfloat16, ignored=ignored)
    check(cuda, 600, 300, 64, torch.float32, "none", ignored=ignored)


def test_left_out_rows_are_not_read(cuda):
    x, w, t, b = inputs(500, 300, 72, ignored=0.5)

    def run():
        ts = [v.float().to(cuda).requires_grad_() for v in (x, w, b)]
        loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2])
        return loss, *torch.autograd.grad(loss, ts)

    want = run()
    x[t == -100] = math.nan
    got = run()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert bool((got[1][(t == -100).to(cuda)] == 0).all())


def test_pieces(cuda):
    """More than half a gigabyte of probabilities: several pieces of the vocabulary, the last
    one ragged, against one row block at a time in float64 on the GPU."""
    N, V, D = 6000, 60001, 64
    r = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(N, D, device=cuda, generator=r).bfloat16().requires_grad_()
    w = (torch.randn(V, D, device=cuda, generator=r) * 0.2).bfloat16().requires_grad_()
    t = torch.randint(0, V, (N,), device=cuda, generator=r)
    loss = linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    xd, wd = x.detach().double(), w.detach().double()
    total, wdx, wdw = 0.0, [], torch.zeros_like(wd)
    for at in range(0, N, 1000):
        l = xd[at : at + 1000] @ wd.t()
        lse = l.logsumexp(-1)
        rows = torch.arange(l.shape[0], device=cuda)
        total += float((lse - l[rows, t[at : at + 1000]]).sum())
        d = (l - lse[:, None]).exp()
        d[rows, t[at : at + 1000]] -= 1
        wdx.append(d @ wd)
        wdw += d.t() @ xd[at : at + 1000]
    assert abs(loss.item() / total - 1) <= 1e-5
    assert off(dx, torch.cat(wdx)) <= TOL[torch.bfloat16]
    assert off(dw, wdw) <= TOL[torch.bfloat16]


def _columns(t):
    wide = torch.zeros(t.shape[0], t.shape[1] + 24, dtype=t.dtype, device=t.device)
    wide[:, 8:-16] = t
    return wide[:, 8:-16]


@pytest.mark.parametrize("layout", [_columns, lambda t: t.t().contiguous().t()])
def test_strides(cuda, layout):
    check(cuda, 70, 90, 64, torch.bfloat16, layout=layout)
    check(cuda, 70, 90, 50, torch.float32, layout=layout)


def test_target_outside_the_vocabulary(cuda):
    x, w, t, b = inputs(20, 30, 16, ignored=0)
    ts = [v.float().to(cuda) for v in (x, w, b)]
    for bad in (-1, 30, 2**40, -(2**40)):
        t[3] = bad
        each = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2], reduction="none")
        assert bool(each[3].isnan()) and int(each.isnan().sum()) == 1


def test_extreme_logits(cuda):
    """Logits in the thousands: one-hot and tied softmaxes, no overflow."""
    x = torch.tensor([[100.0, 0.0], [0.0, 100.0], [-100.0, -100.0]], device=cuda)
    w = torch.tensor([[50.0, 0.0], [0.0, 50.0], [50.0, 0.0]], device=cuda)
    t = torch.tensor([0, 1, 1], device=cuda)
    for v in (x, w):
        v.requires_grad_()
    loss = linear_cross_entropy(x, w, t, reduction="none")
    want = torch.tensor([math.log(2), 0.0, math.log(3)], device=cuda)
    assert torch.allclose(loss, want, atol=1e-6)
    dx, dw = torch.autograd.grad(loss.sum(), (x, w))
    _, wx, ww, _ = plain(x.detach().double(), w.detach().double(), t, None, "sum",
                         torch.ones((), device=cuda))
    assert torch.allclose(dx.double(), wx, atol=1e-4) and torch.allclose(dw.double(), ww, atol=1e-4)


def test_only_some_gradients(cuda):
    x, w, t, b = inputs(90, 120, 48)
    want = plain(x.float().double(), w.float().double(), t, b.float().double())
    for asked in ((0,), (1,), (2,), (0, 2)):
        ts = [v.float().to(cuda).requires_grad_(i in asked) for i, v in enumerate((x, w, b))]
        loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2])
        for i, g in zip(asked, torch.autograd.grad(loss, [ts[i] for i in asked])):
            assert off(g, want[1 + i]) <= TOL[torch.float32]


def test_same_on_every_run(cuda):
    x, w, t, b = inputs(700, 900, 256)
    ts = [v.bfloat16().to(cuda).requires_grad_() for v in (x, w, b)]

    def once():
        loss = linear_cross_entropy(ts[0], ts[1], t.to(cuda), ts[2])
        return loss, *torch.autograd.grad(loss, ts)

    assert all(torch.equal(p, q) for p, q in zip(once(), once()))


def test_other_stream_and_graph(cuda):
    x, w, t, b = inputs(300, 700, 128)
    ts = [v.float().to(cuda).requires_grad_() for v in (x, w, b)]
    t = t.to(cuda)

    def step():
        loss = linear_cross_entropy(ts[0], ts[1], t, ts[2])
        grads = torch.autograd.grad(loss, ts)
        return loss.detach(), *grads

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            ts[0].mul_(0.9)
            t[i * 7 : i * 7 + 5] = -100  # another number of rows that count
        graph.replay()
        got = [v.clone() for v in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), i


def test_declines(cuda, monkeypatch):
    x, w, t, b = inputs(5, 6, 7)
    args = [v.to(cuda) for v in (x, w, t, b)]
    with pytest.raises(RuntimeError, match="float64"):
        linear_cross_entropy(*args)
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    with pytest.warns(UserWarning, match="linear_cross_entropy"):
        loss = linear_cross_entropy(*args)
    assert abs(float(loss) - float(plain(x, w, t, b)[0])) <= 1e-12
