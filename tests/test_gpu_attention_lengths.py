"""Lengths of any integer type and size, as the eager body takes them: at most the sequences' length
counts, below 0 is 0."""

import pytest
import torch

from mingru_amd import linear_attention
from tests.test_linear_attention import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, large", [(torch.int64, 2**63 - 1), (torch.int64, 2**32), (torch.int64, 2**40 + 7),
                                          (torch.int32, 2**31 - 1), (torch.int16, 2**15 - 1),
                                          (torch.uint8, 255), (torch.uint32, 2**32 - 1)])
def test_large_lengths(cuda, monkeypatch, dtype, large):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    ts = [t.float().to(cuda) for t in inputs(3, 70, 2, 1, 16, 16)]
    want = linear_attention(*ts, torch.tensor([70, 0, 5], device=cuda, dtype=torch.int32))
    low = 0 if dtype == torch.uint8 else torch.iinfo(dtype).min
    got = linear_attention(*ts, torch.tensor([large, low, 5], device=cuda, dtype=dtype))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
