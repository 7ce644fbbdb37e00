"""The paged cache's operators on the GPU with an empty table or a cache without pages: the kernels'
manner, NaN for what has no place, without a look at the device's values from the host."""

import math

import pytest
import torch

from mingru_amd import paged_attention_step, paged_cache_append
from tests.test_paged_cache import append_plain

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.int8])
@pytest.mark.parametrize("N, M", [(0, 3), (5, 0), (0, 0)])
def test_attend(cuda, dtype, kind, N, M):
    new = lambda *s: torch.ones(*s, dtype=dtype, device=cuda)  # noqa: E731
    lengths = torch.tensor([0, 1, -3, 7], dtype=kind, device=cuda)
    for window in (None, 2):
        o = paged_attention_step(new(4, 6, 8), new(N, 2, 4, 8), new(N, 2, 4, 5),
                                 torch.zeros(4, M, dtype=kind, device=cuda), lengths, window=window)
        assert o.shape == (4, 6, 5) and o.dtype == dtype and o.is_contiguous()
        assert bool(torch.isnan(o[1::2]).all()) and not bool(o[::2].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.int8])
@pytest.mark.parametrize("N, M", [(0, 3), (5, 0), (0, 0)])
@pytest.mark.parametrize("padded", [False, True])
def test_append(cuda, dtype, kind, N, M, padded):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    s = dict(k=r(3, 5, 2, 8), v=r(3, 5, 2, 6), k_cache=r(N, 2, 4, 8), v_cache=r(N, 2, 4, 6),
             pages=torch.tensor([[0, -1, 3]] * 3)[:, :M].to(kind), start=torch.tensor([0, 2, -1]),
             q=r(3, 5, 4, 8), lengths=torch.tensor([5, 0, 3]) if padded else None,
             frequencies=torch.tensor([1.0, 0.1]))
    want, kc, vc = append_plain(**s)
    dev = {n: t if t is None else t.to(cuda) for n, t in s.items()}
    q = paged_cache_append(**dev).double().cpu()
    assert torch.equal(torch.isnan(q), torch.isnan(want))
    # Of values up to about 3, as in the operator's own tests: 2^-21 and the result's rounding.
    bound = 2.0**-21 * 9 + torch.finfo(dtype).eps / 2 * torch.nan_to_num(want).abs()
    assert bool((torch.nan_to_num(q - want).abs() <= bound).all())
    assert torch.equal(dev["k_cache"].cpu().double(), kc) and torch.equal(dev["v_cache"].cpu().double(), vc)
    assert paged_cache_append(**{**dev, "q": None}) is None


def test_in_a_graph(cuda):
    """Captured, so that a look from the host would fail, and replayed on other lengths."""
    new = lambda *s: torch.ones(*s, device=cuda)  # noqa: E731
    pages, at = torch.zeros(2, 0, dtype=torch.int64, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    lengths = torch.tensor([0, 1], device=cuda)
    q, kc, vc = new(2, 1, 4, 8), new(3, 2, 4, 8), new(3, 2, 4, 6)

    def step():
        turned = paged_cache_append(q[:, :, :2], q[:, :, :2, :6], kc, vc, pages, at, q=q, lengths=lengths)
        return turned, paged_attention_step(q[:, 0], kc, vc, pages, lengths)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for values in ([0, 1], [1, 0], [0, 0], [2, 5]):
        lengths.copy_(torch.tensor(values))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(torch.nan_to_num(a, math.pi), torch.nan_to_num(b, math.pi))
            assert torch.equal(torch.isnan(a).flatten(1).all(1).cpu(), torch.tensor(values) > 0)
