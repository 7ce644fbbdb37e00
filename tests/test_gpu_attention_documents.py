"""The gradient of the decays in packed documents: nothing after a start depends on a decay before it,
so a document's gradient is as exact as it is alone, and 0 where its own upstream gradient is.

Tolerance, of each document's norm: the decays' gradient of fp32 inputs in
test_gpu_linear_attention.py, 4 * 6 * sqrt(128) * 2^-24; bf16 inputs are exact in the products that
feed it, and its other terms are sums in fp32 of three planes of 8 bits: the same."""

import math

import pytest
import torch

from mingru_amd import linear_attention
from tests.test_gpu_attention_planes import on_device
from tests.test_linear_attention import inputs

pytestmark = pytest.mark.gpu

TOL = 4 * 6 * math.sqrt(128) * 2.0**-24


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def packed(B, T, H, Hk, dk, dv, starts, dtype, seed=0):
    q, k, v, g, h = inputs(B, T, H, Hk, dk, dv, seed, documents=False)
    for i, at in enumerate(starts):
        g[:, at] = (-math.inf, -1e30, -200.0)[i % 3]
    return [t.to(dtype) for t in (q, k, v)] + [g.float(), h.float()]


STARTS = [1, 63, 64, 65, 128, 200, 201, 390, 511, 640]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk, dv", [(16, 24), (128, 128)])
def test_documents_without_an_upstream_gradient(cuda, dtype, dk, dv):
    T, ends = 700, [*STARTS, 700]
    ts = [t.to(cuda).requires_grad_() for t in packed(2, T, 2, 1, dk, dv, STARTS, dtype)]
    o, S = linear_attention(*ts)
    for n in range(len(STARTS) + 1):  # only document n has one
        lo, hi = (0 if n == 0 else STARTS[n - 1]), ends[n]
        do = torch.zeros_like(o)
        do[:, lo:hi] = 100 * torch.randn(2, hi - lo, 2, dv, device=cuda).to(dtype)
        dg, = torch.autograd.grad(o, ts[3], do, retain_graph=True)
        dg[:, lo + 1 : hi] = 0  # its first token's decay is what starts it over, 0 as well
        if n == 0:
            dg[:, 0] = 0
        assert float(dg.abs().max()) == 0, n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B, T, H, Hk, dk, dv, starts", [
    (2, 700, 2, 1, 16, 24, STARTS),
    (1, 400, 2, 2, 128, 128, [100, 130, 390]),
    # As many pairs as the chip holds at once: one segment, gone through in blocks of 1024.
    (128, 2500, 4, 4, 4, 4, [10, 451, 452, 476, 1475, 1476, 1477, 1540, 2499]),
])
def test_gradients_of_many_sizes(cuda, dtype, B, T, H, Hk, dk, dv, starts):
    vals = packed(B, T, H, Hk, dk, dv, starts, dtype)
    bounds = [0, *starts, T]
    r = torch.Generator().manual_seed(3)
    do = torch.randn(B, T, H, dv, generator=r)
    for n, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        do[:, lo:hi] *= (1.0, 1e5, 1e-5, 1e2)[n % 4]
    do = do.to(dtype)
    dh = torch.randn(B, H, dk, dv, generator=r)
    ref = [t.to(cuda).double().requires_grad_() for t in vals]
    up = (do.to(cuda).double(), dh.to(cuda).double())
    want = torch.autograd.grad(on_device(*ref), ref, up)[3].cpu()
    dev = [t.to(cuda).requires_grad_() for t in vals]
    got = torch.autograd.grad(linear_attention(*dev), dev, (do.to(cuda), dh.to(cuda)))[3]
    got = got.double().cpu()
    errors = {}
    for lo, hi in zip(bounds, bounds[1:]):
        a, b = got[:, lo:hi], want[:, lo:hi]
        if hi - lo == 1 and lo:
            assert float(a.abs().max()) == 0
            continue
        errors[lo] = float((a - b).norm() / b.norm().clamp(min=1e-300))
    print({n: f"{e:.1e}" for n, e in errors.items()}, flush=True)
    assert max(errors.values()) <= TOL, errors
