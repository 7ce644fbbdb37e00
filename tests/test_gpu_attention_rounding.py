"""bf16 outputs of ``linear_attention`` are as near to the exact ones as bf16 allows: the rounding of the
result is the only one that counts.

Tolerance: the 2-norm of the error is at most 1.1 times that of the exact result's own rounding.
What feeds the outputs holds 16 bits or more: 2^-17 against 2^-9, and fp32 sums."""

import pytest
import torch

from mingru_amd import linear_attention
from tests.test_gpu_attention_planes import off, on_device
from tests.test_linear_attention import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B, T, H, Hk, dk, dv", [(2, 300, 4, 2, 64, 64), (1, 700, 2, 2, 128, 128),
                                                 (64, 200, 4, 4, 128, 128), (2, 333, 3, 1, 48, 80),
                                                 (1, 500, 2, 1, 100, 37), (2, 129, 2, 2, 128, 64)])
@pytest.mark.parametrize("documents", [False, True])
def test_one_rounding(cuda, monkeypatch, B, T, H, Hk, dk, dv, documents):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    vals = inputs(B, T, H, Hk, dk, dv, seed=T, documents=documents)
    vals = [t.bfloat16() for t in vals[:3]] + [t.float() for t in vals[3:]]
    r = torch.Generator().manual_seed(5)
    do = torch.randn(B, T, H, dv, generator=r).bfloat16().to(cuda)
    dh = torch.randn(B, H, dk, dv, generator=r).to(cuda)
    ref = [t.to(cuda).double().requires_grad_() for t in vals]
    want = on_device(*ref)
    wgrads = torch.autograd.grad(want, ref[:3], (do.double(), dh.double()))
    dev = [t.to(cuda).requires_grad_() for t in vals]
    got = linear_attention(*dev)
    grads = torch.autograd.grad(got, dev[:3], (do, dh))
    errors = {}
    for n, a, b in zip(("o", "dq", "dk", "dv"), (got[0], *grads), (want[0], *wgrads)):
        assert a.dtype == torch.bfloat16
        errors[n] = off(a, b) / off(b.detach().bfloat16(), b)
    print({n: round(e, 4) for n, e in errors.items()}, flush=True)
    assert max(errors.values()) <= 1.1, errors
