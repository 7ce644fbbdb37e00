"""``linear_cross_entropy`` where one thread, wave or workgroup a row, weight or tile would pass the 2^32
threads that a launch can have."""

import pytest
import torch

from mingru_amd import linear_cross_entropy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    yield
    torch.cuda.empty_cache()


def test_many_weights(cuda):
    """2^26 and a few rows of weights that are packed."""
    V = (1 << 26) + 5
    r = torch.Generator(device=cuda).manual_seed(0)
    w = torch.randn(V, 1, device=cuda, generator=r).bfloat16()
    x = torch.tensor([[0.5], [-2.0], [1.0]], device=cuda).bfloat16()
    t = torch.tensor([V - 1, 3, V // 2], device=cuda)
    got = linear_cross_entropy(x, w, t, reduction="none")
    l = x.double() @ w.double().t()
    want = l.logsumexp(-1) - l.gather(1, t[:, None])[:, 0]
    assert float(((got - want).abs() / want).max()) <= 1e-5


def test_many_tiles(cuda):
    """More than 2^24 tiles of logits."""
    N, V, D = 1 << 20, (1 << 19) + 256, 8
    r = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(N, D, device=cuda, generator=r).bfloat16()
    w = torch.randn(V, D, device=cuda, generator=r).bfloat16()
    t = torch.randint(0, V, (N,), device=cuda, generator=r)
    whole = linear_cross_entropy(x, w, t, reduction="none")
    half = N // 2
    for rows in (slice(0, half), slice(half, N)):
        assert torch.equal(whole[rows], linear_cross_entropy(x[rows], w, t[rows], reduction="none"))


def test_many_rows(cuda):
    """2^28 and a few rows."""
    N = (1 << 28) + 70
    r = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(N, 1, device=cuda, generator=r).bfloat16()
    w = torch.tensor([[0.5], [-1.5], [1.0]], device=cuda).bfloat16()
    t = torch.randint(0, 3, (N,), device=cuda, generator=r)
    loss = linear_cross_entropy(x, w, t, reduction="none")
    for rows in (slice(0, 5000), slice(1 << 27, (1 << 27) + 5000), slice(N - 5000, N)):
        l = x[rows].double() @ w.double().t()
        want = l.logsumexp(-1) - l.gather(1, t[rows, None])[:, 0]
        assert float((loss[rows] - want).norm() / want.norm()) <= 1e-5
