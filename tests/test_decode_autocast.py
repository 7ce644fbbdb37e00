"""The decode operators' eager bodies under autocast: what they hold in 32 bits stays so."""

import pytest
import torch

from mingru_amd import beam_select, paged_attention_step, paged_cache_append
from tests.test_paged_cache import append_inputs, attend_inputs


@pytest.fixture(autouse=True)
def _eager(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "eager")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_results_are_the_same(dtype):
    a = attend_inputs(3, 4, 2, 64, 48, 4, 20, dtype=dtype)
    g = torch.Generator().manual_seed(0)
    logits, scores = torch.randn(2, 3, 50, generator=g).to(dtype), torch.zeros(2, 3)

    def run():
        s = append_inputs(2, 3, 2, 1, 8, 4, 2, 3, 4, dtype=dtype)
        q = paged_cache_append(**s)
        return [paged_attention_step(**a), q, s["k_cache"], s["v_cache"], *beam_select(logits, scores, 4)]

    want = run()
    for half in (torch.bfloat16, torch.float16):
        with torch.autocast("cpu", dtype=half):
            got = run()
        assert all(x.dtype == y.dtype and torch.equal(x, y) for x, y in zip(got, want))
