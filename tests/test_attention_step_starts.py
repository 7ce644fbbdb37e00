"""A step that starts a document sees nothing of the state before, whatever it holds: infinities and
NaN (a recycled slot) do not reach past it, and it starts over wherever the pass does, at factors
below the smallest normal float.  Results are compared with those from a state of 0, exactly."""

import math

import pytest
import torch

from mingru_amd import linear_attention, linear_attention_step
from tests.test_linear_attention import inputs


@pytest.mark.parametrize("junk", [math.nan, math.inf, 3e38])
@pytest.mark.parametrize("g0", [-math.inf, -1e30, -120.0, -88.0])
def test_step(junk, g0):
    q, k, v = (t[:, 0].float() for t in inputs(2, 1, 4, 2, 5, 3)[:3])
    g = torch.full((2, 4), g0)
    got = linear_attention_step(q, k, v, g, torch.full((2, 4, 5, 3), junk))
    want = linear_attention_step(q, k, v, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("junk", [math.nan, math.inf, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g0", [-math.inf, -1e30, -120.0, -88.0])
def test_step_on_the_gpu(cuda, monkeypatch, junk, dtype, g0):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    q, k, v, g, _ = (t.to(cuda) for t in inputs(2, 1, 4, 2, 24, 37))
    q, k, v = (t[:, 0].to(dtype) for t in (q, k, v))
    g = torch.full((2, 4), g0, device=cuda)
    h = torch.full((2, 4, 24, 37), junk, device=cuda)
    got = linear_attention_step(q, k, v, g, h)
    want = linear_attention_step(q, k, v, g)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_step_is_the_pass_at_the_smallest_factors(cuda, monkeypatch):
    """Just above and below the smallest normal float, with a state that makes it visible."""
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    q, k, v, _, _ = (t.float().to(cuda) for t in inputs(1, 1, 2, 2, 16, 16))
    h = torch.full((1, 2, 16, 16), 3e37, device=cuda)
    for g0 in (-87.0, -87.3, -87.4, -88.0, -90.0, -103.0, -104.0):
        g = torch.full((1, 2), g0, device=cuda)
        o, S = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, h)
        wo, wS = linear_attention(q, k, v, g[:, None], h)
        # Exponents of size 126 rounded to 2^-18 of 1, each way; sums of 16 terms of either sign.
        assert float((S - wS).norm()) <= 2.0**-16 * float(wS.norm()), g0
        assert float((o - wo[:, 0]).norm()) <= 2.0**-14 * float(wo.norm()), g0
