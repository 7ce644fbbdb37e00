"""``paged_attention_step`` where no token is attended to and outputs are many."""

import pytest
import torch

from mingru_amd import paged_attention_step

pytestmark = pytest.mark.gpu


def test_zeros_past_2_to_31_elements_of_a_sequence(cuda, monkeypatch):
    """2^23 heads of 256: a sequence's outputs are as many as 31 bits no longer count."""
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    H, dv = 2**23, 256
    filled = torch.full((1, H, dv), 3.0, dtype=torch.bfloat16, device=cuda)
    del filled  # its memory is the next one of its size
    new = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=cuda)  # noqa: E731
    o = paged_attention_step(new(1, H, 1), new(1, 1, 16, 1), new(1, 1, 16, dv),
                             torch.zeros(1, 1, dtype=torch.int64, device=cuda),
                             torch.zeros(1, dtype=torch.int64, device=cuda))
    assert not bool(o.view(-1).view(torch.int32).any())
