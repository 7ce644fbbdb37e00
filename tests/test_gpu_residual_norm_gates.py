"""The gates of ``residual_norm`` in fp32, element by element, over all that is representable: relative to
the result, so that a nearly closed gate counts as well.

Tolerance: an exponential and a reciprocal of 1 ulp (2^-23) each, the sum between them 2^-24 and
the correction's product 2^-24, gate times row 2^-24: 2 * 2^-23 + 3 * 2^-24 = 4.2e-7."""

import math

import pytest
import torch

from mingru_amd import residual_norm

pytestmark = pytest.mark.gpu

TOL = 2 * 2.0**-23 + 3 * 2.0**-24


@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("D", [8, 7])
def test_gates(cuda, monkeypatch, act, D):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    x = torch.cat([torch.linspace(-86, 86, 1 << 17), torch.linspace(-1e-3, 1e-3, 1 << 12)])
    x = x[: len(x) // D * D].view(-1, D).to(cuda)
    got = residual_norm(torch.ones_like(x), gate=x, gate_act=act, pre="none").double()
    want = torch.sigmoid(x.double()) * (x.double() if act == "silu" else 1)
    live = want != 0
    assert float(((got - want).abs() / want.abs())[live].max()) <= TOL
    assert bool((got[~live] == 0).all())


def test_gates_at_the_ends(cuda, monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    x = torch.tensor([[math.inf, -math.inf, math.nan, 1e30, -1e30, 200.0, -200.0, -0.0]], device=cuda)
    for act in ("sigmoid", "silu"):
        got = residual_norm(torch.ones_like(x), gate=x, gate_act=act, pre="none")
        want = torch.sigmoid(x) * (x if act == "silu" else 1)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), act
