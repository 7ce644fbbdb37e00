"""Where a document starts nothing of the state before is seen, whatever that state holds: infinities
and NaN in it (a recycled slot) do not reach past a start, in the pass or its gradients.  Results
are compared with those from a state of 0, exactly."""

import math

import pytest
import torch

from mingru_amd import linear_attention
from tests.test_linear_attention import inputs


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("T, start", [(1, 0), (30, 0), (150, 0), (150, 31), (150, 64), (150, 140)])
def test_pass(junk, T, start):
    q, k, v, g, h = (t.float() for t in inputs(2, T, 2, 1, 5, 3, documents=False))
    g[:, start] = -math.inf
    r = torch.Generator().manual_seed(0)
    do, dh = torch.randn(2, T, 2, 3, generator=r), torch.randn(2, 2, 5, 3, generator=r)
    do[:, :start] = 0

    def run(h0):
        ts = [t.detach().clone().requires_grad_() for t in (q, k, v, g, h0)]
        o, S = linear_attention(*ts)
        grads = torch.autograd.grad((o, S), ts, (do, dh))
        return o[:, start:], S, *(t[:, start:] for t in grads[:4]), grads[4]

    for n, a, b in zip(("o", "S", "dq", "dk", "dv", "dg", "dh0"), run(torch.full_like(h, junk)),
                       run(torch.zeros_like(h))):
        assert torch.equal(a, b), n


@pytest.mark.gpu
@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, start", [(1, 0), (40, 0), (300, 0), (300, 31), (300, 64), (300, 200)])
@pytest.mark.parametrize("dk, dv", [(24, 37), (128, 128)])
def test_pass_on_the_gpu(cuda, monkeypatch, junk, dtype, T, start, dk, dv):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    q, k, v, g, h = (t.to(cuda) for t in inputs(2, T, 2, 1, dk, dv, documents=False))
    q, k, v, g, h = q.to(dtype), k.to(dtype), v.to(dtype), g.float(), h.float()
    g[:, start] = -math.inf
    r = torch.Generator(device=cuda).manual_seed(0)
    do = torch.randn(2, T, 2, dv, device=cuda, generator=r).to(dtype)
    do[:, :start] = 0  # tokens before the start do see that state
    dh = torch.randn(2, 2, dk, dv, device=cuda, generator=r)

    def run(h0):
        ts = [t.detach().clone().requires_grad_() for t in (q, k, v, g, h0)]
        o, S = linear_attention(*ts)
        grads = torch.autograd.grad((o, S), ts, (do, dh))
        return o[:, start:], S, *(t[:, start:] for t in grads[:4]), grads[4]

    bad = torch.zeros_like(h)
    bad[0] = junk
    bad[1, 0, 0, 0] = junk
    for n, a, b in zip(("o", "S", "dq", "dk", "dv", "dg", "dh0"), run(bad), run(torch.zeros_like(h))):
        assert torch.equal(a, b), n
