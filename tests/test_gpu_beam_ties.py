"""``beam_select`` kernels on beams of equal logits: whatever a row's address, its sum is the same, so that
candidates of equal scores come by the lower beam, then by the lower token."""

import math

import pytest
import torch

from mingru_amd import beam_select

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, K, V, width", [
    (1, 4, 50257, 4), (3, 8, 50257, 8), (2, 16, 32771, 32), (5, 6, 3001, 64), (1, 256, 3001, 64),
    (4, 3, 2049, 20), (7, 5, 5, 9), (9, 4, 7, 20), (3, 3, 1, 3), (2, 64, 9, 64), (300, 2, 17, 34)])
def test_equal_beams(cuda, dtype, B, K, V, width):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, 1, V, generator=g).mul(4).to(dtype).expand(-1, K, -1)
    scores = -torch.rand(B, 1, generator=g).expand(-1, K)
    # Of equal sums, scores order as logits do.
    order = torch.sort(x.double().flatten(1), dim=-1, descending=True, stable=True)[1][:, :width]
    score, parent, token = beam_select(x.contiguous().to(cuda), scores.contiguous().to(cuda), width)
    assert torch.equal(parent.cpu(), order // V) and torch.equal(token.cpu(), order % V)
    log = torch.log_softmax(x.double(), -1) + scores.double()[..., None]
    want = log.flatten(1).gather(1, order)
    # A sum's error is 2^-22 of it at most, a result's rounding 2^-24 of it.
    assert not bool(((score.double().cpu() - want).abs() > 2.0**-22 + 2.0**-24 * want.abs()).any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 3, 4, 7, 8, 9, 63, 2047, 2048, 2049, 2055, 3001, 50257])
def test_results_do_not_depend_on_the_address(cuda, dtype, V):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(2, 3, V, generator=g).mul(4).to(dtype).to(cuda)
    scores = -torch.rand(2, 3, generator=g).to(cuda)
    width = min(8, 3 * V)
    want = beam_select(x, scores, width)
    for at in range(1, 9):
        wide = torch.full((2, 3, V + 16), math.nan, dtype=dtype, device=cuda)
        wide[..., at : at + V] = x
        got = beam_select(wide[..., at : at + V], scores, width)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), at


@pytest.mark.parametrize("dtype", TYPES)
def test_neighbours_do_not_count(cuda, dtype):
    """What lies before and behind a row has no part in it."""
    for V in (1, 2, 5, 11, 2049, 4093):
        room = torch.full((V + 32,), math.inf, dtype=dtype, device=cuda)
        g = torch.Generator().manual_seed(V)
        x = torch.randn(V, generator=g).to(dtype)
        for at in (0, 1, 5, 16):
            room.fill_(math.inf)
            room[at : at + V] = x.to(cuda)
            width = min(V, 64)
            score, parent, token = beam_select(room[at : at + V].view(1, 1, V),
                                               torch.zeros(1, 1, device=cuda), width)
            want = torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][:width]
            assert torch.equal(token[0].cpu(), want) and not bool(parent.any())
            log = torch.log_softmax(x.double(), -1)[want]
            assert not bool(((score[0].double().cpu() - log).abs() > 2.0**-22 + 2.0**-24 * log.abs()).any())
