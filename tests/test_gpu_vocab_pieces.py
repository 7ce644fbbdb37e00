"""``linear_cross_entropy`` over several pieces of the vocabulary, with a bias, left-out rows and rows'
own upstream gradients, against one row block at a time in float64 on the GPU.  Tolerances as for
one piece: 1e-5 of a gradient's norm in fp32, two roundings to 8 bits in bf16."""

import math

import pytest
import torch

from mingru_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2 * 2.0**-8}


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def off(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("dtype, V", [(torch.float32, 60001), (torch.bfloat16, 120001)])
def test_pieces(cuda, dtype, V, reduction):
    N, D = 5000, 72
    r = torch.Generator(device=cuda).manual_seed(0)
    n = lambda *s: torch.randn(*s, device=cuda, generator=r)  # noqa: E731
    x, w, b = n(N, D).to(dtype), (n(V, D) * (1.5 / math.sqrt(D))).to(dtype), (0.5 * n(V)).to(dtype)
    t = torch.randint(0, V, (N,), device=cuda, generator=r)
    t[torch.rand(N, device=cuda, generator=r) < 0.3] = -100
    keep = t != -100
    up = n(N) if reduction == "none" else n(1)[0]
    ts = [v.requires_grad_() for v in (x, w, b)]
    loss = linear_cross_entropy(x, w, t, b, reduction=reduction)
    dx, dw, db = torch.autograd.grad(loss, ts, up)
    xd, wd, bd = (v.detach().double() for v in ts)
    g = (up.double() if reduction == "none" else up.double() / keep.sum()) * keep
    each, wdx, wdw, wdb = [], [], torch.zeros_like(wd), torch.zeros_like(bd)
    for at in range(0, N, 1000):
        rows = slice(at, at + 1000)
        l = xd[rows] @ wd.t() + bd
        at_t = torch.where(keep[rows], t[rows], 0)[:, None]
        lse = l.logsumexp(-1)
        each.append((lse - l.gather(1, at_t)[:, 0]) * keep[rows])
        d = (l - lse[:, None]).exp_()
        d.scatter_add_(1, at_t, torch.full_like(at_t, -1.0, dtype=d.dtype))
        d *= g[rows, None]
        wdx.append(d @ wd)
        wdw += d.t() @ xd[rows]
        wdb += d.sum(0)
    each, wdx = torch.cat(each), torch.cat(wdx)
    want = each if reduction == "none" else each.sum() / keep.sum()
    errors = {"loss": off(loss.detach(), want) / 1e-5, "dx": off(dx, wdx) / TOL[dtype],
              "dw": off(dw, wdw) / TOL[dtype], "db": off(db, wdb) / TOL[dtype]}
    print({k: round(e, 3) for k, e in errors.items()}, flush=True)
    assert max(errors.values()) <= 1, errors
    assert bool((dx[~keep] == 0).all())
