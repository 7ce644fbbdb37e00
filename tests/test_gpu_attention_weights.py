"""``paged_attention_step`` where small weights carry the result, against the definition in float64."""

import math

import pytest
import torch

from mingru_amd import paged_attention_step
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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk, dv, P", [(64, 64, 16), (128, 128, 16), (256, 256, 7)])
def test_weights_keep_their_bits_where_values_cancel(cuda, dtype, dk, dv, P):
    """Four tokens whose weighted values sum to nearly 0, so that the weights' own rounding shows and the
    result's does not.  S is the sum of the values' weighted magnitudes.

    Scores are one exact product each, 1 at most, taken times a scale of three roundings (its own, its
    product with log2 e and theirs) and off by one more from the largest: 4 * 1.45 * ln 2 * 2^-24 =
    4 * 2^-24 of a weight.  Its exponential is 2 * 2^-24 off, its summands (fp16's two) 4 * 2^-24, and
    12 additions, each of S at most, 12 * 2^-24 of that; the sum of weights scales a result that is
    nearly 0.  22 * 2^-24 < 2^-19 of S in all, where two summands of bf16 lose up to 2^-17."""
    B, H, Hk = 64, 16, 16
    s = attend_inputs(B, H, Hk, dk, dv, P, -(-4 // P), dtype=dtype)
    g = torch.Generator().manual_seed(dk)
    s["lengths"] = torch.full((B,), 4)
    s["q"], s["k_cache"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k_cache"])
    s["q"][..., 3] = 1.0
    scores = torch.rand(B, H, 4, generator=g).to(dtype)
    p = torch.softmax(scores.double(), -1)
    v = torch.empty(B, H, 4, dv, dtype=dtype)
    v[:, :, 0] = (1 + torch.rand(B, H, dv, generator=g)).to(dtype)
    for i in range(1, 4):  # each takes off what is left, to its type's rounding
        left = (p[:, :, :i, None] * v[:, :, :i].double()).sum(2)
        v[:, :, i] = (-left / p[:, :, i, None]).to(dtype)
    for b in range(B):
        for j in range(4):
            page, slot = s["pages"][b, j // P], j % P
            s["k_cache"][page, :, slot, 3] = scores[b, :, j]
            s["v_cache"][page, :, slot] = v[b, :, j]
    want = (p[..., None] * v.double()).sum(2)
    size = (p[..., None] * v.double().abs()).sum(2)
    got = paged_attention_step(**{n: t.to(cuda) for n, t in s.items()}, scale=1.0).double().cpu()
    bound = 2.0**-19 * size + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / size).max() * 2**24)
