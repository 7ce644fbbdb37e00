"""``paged_attention_step`` where small weights carry the result, against the definition in float64."""

import math

import pytest
import torch

from tests.test_gpu_paged_cache import TYPES, check_attend
from tests.test_paged_cache import attend_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("octaves", [10, 16, 22, 26, 30])
@pytest.mark.parametrize("n, heavy", [(20, 0), (100, 0), (100, 99), (5000, 4999),
                                      (65536, 0), (65536, 40000)])
def test_weights_far_below_the_largest(cuda, dtype, octaves, n, heavy):
    """One token has nearly all weight and a value of 0, so that the rest of them is the result: through
    one share of the work, and through the join of many.  Scores are one exact product each; forming
    a weight from up to 30 octaves takes three roundings of 2^-24 of those, 62 * 2^-24 of the weight,
    less than the 128 * 2^-24 that the tolerance counts.  Values are large enough for results that are
    normal numbers of every type."""
    s = attend_inputs(1, 6, 2, 64, 48, 16, -(-n // 16), dtype=dtype)
    g = torch.Generator().manual_seed(n + octaves)
    s["lengths"] = torch.tensor([n])
    s["q"], s["k_cache"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k_cache"])
    s["q"][..., 5] = 1.0
    s["k_cache"][..., 5] = torch.rand(s["k_cache"].shape[:-1], generator=g)
    s["v_cache"] = (2.0**14 * (1 + 2 * torch.rand(s["v_cache"].shape, generator=g))).to(dtype)
    page, slot = s["pages"][0, heavy // 16], heavy % 16
    s["k_cache"][page, :, slot, 5] = octaves * math.log(2.0)
    s["v_cache"][page, :, slot] = 0.0
    check_attend(cuda, s, scale=1.0)
