"""``linear_attention`` where one thread or workgroup an element or pair would pass the 2^32
threads that a launch can have: results equal those of parts that are launched apart."""

import pytest
import torch

from mingru_amd import linear_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    yield
    torch.cuda.empty_cache()


def test_many_pairs(cuda):
    """2^22 and a few (sequence, head) pairs of two tokens, with gradients."""
    B, T, H, d = (1 << 20) + 5, 2, 4, 2
    r = torch.Generator(device=cuda).manual_seed(0)
    n = lambda *s: torch.randn(*s, device=cuda, generator=r)  # noqa: E731
    vals = [n(B, T, H, d), n(B, T, H, d), n(B, T, H, d), -n(B, T, H).abs(), n(B, H, d, d)]
    do, dh = n(B, T, H, d), n(B, H, d, d)

    def run(rows):
        ts = [t[rows].detach().requires_grad_() for t in vals]
        out = linear_attention(*ts)
        return *out, *torch.autograd.grad(out, ts, (do[rows], dh[rows]))

    whole = run(slice(None))
    for lo, hi in ((0, 1000), (1 << 19, (1 << 19) + 1000), (B - 1000, B)):
        for a, b in zip(whole, run(slice(lo, hi))):
            assert torch.equal(a[lo:hi], b)


def test_many_elements_of_shared_keys(cuda):
    """2^32 elements of dq and dk, each the sum over the heads that share it."""
    B, T, d = 64, (1 << 19) + 64, 128
    assert B * T * d > 2**32
    r = torch.Generator(device=cuda).manual_seed(0)
    n = lambda *s: torch.randn(*s, device=cuda, generator=r, dtype=torch.bfloat16)  # noqa: E731
    vals = [n(B, T, 1, d), n(B, T, 1, d), n(B, T, 2, 1)]
    g = torch.tensor([-0.01, -0.1], device=cuda)
    do = n(B, T, 2, 1)

    def run(rows):
        ts = [t[rows].detach().requires_grad_() for t in vals]
        o, _ = linear_attention(*ts, g)
        return torch.autograd.grad(o, ts, do[rows])

    whole = run(slice(None))
    # Fewer sequences are cut into other segments: equal but for the rounding of bf16 results.
    for lo in (0, 40, B - 1):
        for a, b in zip(whole, run(slice(lo, lo + 1))):
            a, b = a[lo:lo + 1].float(), b.float()
            assert float((a - b).norm() / b.norm()) <= 2 * 2.0**-8
