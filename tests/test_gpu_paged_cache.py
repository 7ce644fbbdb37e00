"""``paged_cache_append`` and ``paged_attention_step`` kernels against the definition in float64.

Tolerances.  Append, element by element: the angle, reduced to an eighth of a turn or less, is
rounded to fp32 (below 1, by 2^-25 at most); its sine and cosine, two products and a sum are five
more roundings of 2^-24: 2^-21 of the pair's sum of magnitudes is more than all of them.  Then one
rounding of the result, ``eps / 2``.

Attention, as the 2-norm of the difference over that of the result: a score is a sum of up to 256
products, whose rounding is that of as many partial sums of its size, in disorder, sqrt(256) =
16 times 2^-24 of it; scores are up to about 8 here, so a weight is up to 128 * 2^-24 off, its
exponential and the sums of weights and of products a few more: 160 * 2^-24 = 9.6e-6.  Half
types: the same, two summands of a weight (2^-16 of it in bf16) and the result's rounding,
``eps / 2``.
"""

import math

import pytest
import torch

from mingru_amd import paged_attention_step, paged_cache_append
from tests.test_paged_cache import (
    append_inputs,
    append_plain,
    attend_inputs,
    attend_plain,
    poison,
    tables,
)

pytestmark = pytest.mark.gpu

HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TYPES = list(HALF)
ATTEND = {torch.float32: 160 * 2.0**-24, torch.bfloat16: 160 * 2.0**-24 + 2.0**-16 + 2.0**-8,
          torch.float16: 160 * 2.0**-24 + 2.0**-22 + 2.0**-11}


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def to(s, cuda):
    return {n: t.to(cuda) if torch.is_tensor(t) else t for n, t in s.items()}


def check_append(cuda, s, interleaved=False, dev=None):
    dtype = s["k"].dtype
    want = append_plain(**s, interleaved=interleaved)
    dev = to(s, cuda) if dev is None else dev
    before = {n: dev[n].clone() for n in ("k_cache", "v_cache")}
    q = paged_cache_append(**dev, interleaved=interleaved)
    torch.cuda.synchronize()
    for name, a, b in zip("qkv", (q, dev["k_cache"], dev["v_cache"]), want):
        if a is None:
            assert b is None
            continue
        a = a.double().cpu()
        assert torch.equal(torch.isnan(a), torch.isnan(b)), name
        a, b = torch.nan_to_num(a), torch.nan_to_num(b)
        # A pair's magnitudes are at most sqrt(2) times either's length.
        size = 3 * torch.nan_to_num(s[name].double(), 0.0, 0.0, 0.0).abs().max()
        bound = HALF[dtype] * b.abs() + 2.0**-21 * size
        assert bool(((a - b).abs() <= bound).all()), (name, float((a - b).abs().max()))
    for name, old in before.items():  # what no token goes to is left as it was
        new, ref = dev[name], want[1 if name == "k_cache" else 2].to(cuda)
        same = ref == old.double()
        assert bool((new == old)[same].all()), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dk, dv, n", [(128, 128, 64), (64, 80, 16), (80, 48, 20), (256, 32, 0),
                                       (10, 7, 3), (96, 96, 44), (8, 8, 4), (2, 1, 1)])
def test_append_sizes(cuda, dtype, interleaved, dk, dv, n):
    s = append_inputs(3, 5, 4, 2, dk, dv, 4, 6, n, dtype=dtype)
    s["lengths"] = torch.tensor([5, 0, 2])
    check_append(cuda, s, interleaved)


@pytest.mark.parametrize("B, T, H, Hk, P, M", [(1, 1, 1, 1, 1, 1), (1, 100, 0, 3, 7, 20),
                                               (40, 1, 5, 5, 16, 3), (2, 37, 8, 1, 64, 2),
                                               (1, 3, 64, 64, 3, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_shapes(cuda, B, T, H, Hk, P, M, dtype):
    check_append(cuda, append_inputs(B, T, H, Hk, 32, 16, P, M, 16, dtype=dtype))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.int16])
@pytest.mark.parametrize("wide", [torch.float32, torch.float64, torch.bfloat16])
def test_append_integer_and_frequency_types(cuda, kind, wide):
    s = append_inputs(3, 5, 4, 2, 16, 16, 4, 6, 8, dtype=torch.float32)
    s["lengths"] = torch.tensor([5, 0, 2])
    for n in ("pages", "start", "lengths"):
        s[n] = s[n].to(kind)
    s["frequencies"] = s["frequencies"].to(wide)
    check_append(cuda, s)


def test_append_mixed_integers(cuda):
    s = append_inputs(3, 5, 4, 2, 16, 16, 4, 6, 8, dtype=torch.float32)
    s["lengths"], s["pages"] = torch.tensor([5, 0, 2]), s["pages"].int()
    check_append(cuda, s)


@pytest.mark.parametrize("q", [True, False])
def test_append_leaves_out(cuda, q):
    """Negative pages, pages outside of the cache, positions outside of the table."""
    s = append_inputs(4, 6, 2, 1, 8, 8, 2, 4, 4, dtype=torch.float32)
    s["start"] = torch.tensor([0, 2, 5, -3])
    s["pages"][0, 1], s["pages"][1, 2], s["pages"][1, 3] = -1, 19, 2**31 - 1
    if not q:
        s["q"] = None
    check_append(cuda, s)


def test_append_padding_is_not_read(cuda):
    s = append_inputs(2, 3, 2, 1, 8, 8, 2, 4, 4, dtype=torch.bfloat16)
    s["lengths"] = torch.tensor([1, -5])
    for n in "qkv":
        s[n][0, 1:], s[n][1] = math.nan, math.inf
    s["start"][1] = 10**6
    check_append(cuda, s)


@pytest.mark.parametrize("n", [-(2**63), -1, 2**40, 2**63 - 1])
def test_append_lengths_of_64_bits(cuda, n):
    s = append_inputs(2, 5, 2, 1, 8, 8, 2, 4, 4, dtype=torch.float32)
    s["lengths"] = torch.tensor([n, 3])
    check_append(cuda, s)


def test_append_marks_the_caches_as_written(cuda):
    s = to(append_inputs(2, 5, 2, 1, 8, 8, 2, 4, 4, dtype=torch.float32), cuda)
    w = torch.ones((), device=cuda, requires_grad=True)
    y = (w * s["k_cache"]).sum()  # keeps the cache for its gradient
    paged_cache_append(**s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        s = to(append_inputs(2, 5, 2, 1, 8, 8, 2, 4, 4, dtype=torch.float32), cuda)
        paged_cache_append(**s)


def test_append_far_positions(cuda):
    """Angles of positions whose product with a frequency has no more bits in fp32 left."""
    far, n = 3 * 10**6, 64
    s = append_inputs(1, 2, 2, 2, 2 * n, 8, 2, 3, n, dtype=torch.float32)
    s["pages"] = torch.full((1, far // 2 + 2), -1, dtype=torch.int64)
    s["pages"][0, -2:] = torch.tensor([3, 1])
    s["start"] = torch.tensor([far])
    s["frequencies"] = (10000.0 ** (-torch.arange(n) / n)).float()
    check_append(cuda, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_strides(cuda, dtype):
    s = append_inputs(3, 5, 4, 2, 32, 16, 4, 6, 16, dtype=dtype)
    dev = to(s, cuda)
    joined = torch.cat([dev[n].flatten(2) for n in "qkv"], -1)  # slices of one projection
    dev["q"], dev["k"], dev["v"] = (t.unflatten(-1, (-1, d)) for t, d in zip(
        joined.split((128, 64, 32), -1), (32, 32, 16)))
    for n in ("k_cache", "v_cache"):  # (N, P, Hk, d) in memory
        dev[n] = dev[n].transpose(1, 2).contiguous().transpose(1, 2)
    dev["pages"] = torch.stack([dev["pages"]] * 2, -1)[..., 0]
    dev["start"] = torch.stack([dev["start"]] * 2, -1)[:, 0]
    check_append(cuda, s, dev=dev)


def test_append_unaligned(cuda):
    s = append_inputs(3, 5, 4, 2, 32, 16, 4, 6, 16, dtype=torch.bfloat16)
    dev = to(s, cuda)
    for n in ("q", "k", "v", "k_cache", "v_cache"):
        t = torch.empty(dev[n].numel() + 1, dtype=torch.bfloat16, device=cuda)[1:]
        dev[n] = t.view(dev[n].shape).copy_(dev[n])
    check_append(cuda, s, dev=dev)


def test_append_declines(cuda):
    s = append_inputs(3, 5, 4, 2, 32, 16, 4, 6, 16)
    with pytest.raises(RuntimeError, match="float64"):
        paged_cache_append(**to(s, cuda))


def off(a, b):
    return float((a.double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


def check_attend(cuda, s, dev=None, **kw):
    want = attend_plain(**s, **kw)
    got = paged_attention_step(**(to(s, cuda) if dev is None else dev), **kw)
    assert got.shape == want.shape and got.dtype == s["q"].dtype
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got).cpu(), nan)
    zero = s["lengths"] <= 0
    assert not bool(got.cpu()[zero].any())
    got, want = torch.nan_to_num(got), torch.nan_to_num(want)
    assert off(got, want) <= ATTEND[s["q"].dtype], off(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk, dv", [(64, 64), (128, 128), (256, 256), (32, 64), (80, 48), (72, 72),
                                    (192, 128), (100, 7), (1, 1), (65, 129), (16, 200)])
@pytest.mark.parametrize("P", [16, 7])
def test_attend_sizes(cuda, dtype, dk, dv, P):
    s = attend_inputs(5, 6, 2, dk, dv, P, 300 // P, dtype=dtype)
    s["lengths"][:3] = torch.tensor([0, 1, 300 // P * P])
    check_attend(cuda, s)


@pytest.mark.parametrize("H, Hk", [(1, 1), (8, 8), (16, 1), (17, 1), (40, 1), (66, 2), (15, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_heads(cuda, H, Hk, dtype):
    s = attend_inputs(4, H, Hk, 64, 64, 16, 40, dtype=dtype)
    check_attend(cuda, s)


@pytest.mark.parametrize("n", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("P", [1, 4, 16, 33, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_lengths(cuda, n, P, dtype):
    s = attend_inputs(2, 4, 2, 64, 64, P, -(-300 // P), dtype=dtype)
    s["lengths"] = torch.tensor([n, 300 - n])
    check_attend(cuda, s)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 129, 299, 300, 10**6])
@pytest.mark.parametrize("P", [4, 7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attend_windows(cuda, window, P, dtype):
    s = attend_inputs(6, 4, 2, 64, 48, P, 300 // P, dtype=dtype)
    s["lengths"] = torch.tensor([0, 1, 128, 200, 257, 300 // P * P])
    check_attend(cuda, s, window=window)


@pytest.mark.parametrize("B, longest", [(1, 20000), (3, 9000), (70, 700), (300, 200), (1000, 40)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_batches(cuda, B, longest, dtype):
    """Shares that hold many sequences, parts of one, and both; some sequences are empty."""
    s = attend_inputs(B, 4, 2, 64, 64, 16, -(-longest // 16), dtype=dtype)
    s["lengths"][torch.rand(B, generator=torch.Generator().manual_seed(3)) < 0.2] = 0
    s["lengths"][-1] = longest
    check_attend(cuda, s)


@pytest.mark.parametrize("B", [64, 65, 4097, 9000])
def test_attend_many_sequences(cuda, B):
    """More than a wave's lanes find at once, and than their runs; nearly all of them empty."""
    s = attend_inputs(B, 2, 1, 16, 16, 16, 20, dtype=torch.float32)
    some = torch.rand(B, generator=torch.Generator().manual_seed(4)) < 60 / B
    s["lengths"] = torch.where(some, s["lengths"], torch.zeros_like(s["lengths"]))
    s["lengths"][-1] = 320
    check_attend(cuda, s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e", [3, 8, 14, 30, 60])
def test_attend_large_scores(cuda, dtype, e):
    """Scores of 2^(2 e - 3), as exact as sums, so that equal keys share the weight exactly."""
    if dtype == torch.float16 and e > 14:
        pytest.skip("out of the type's range")
    s = attend_inputs(6, 6, 2, 64, 64, 16, 60, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    s["q"] = torch.zeros_like(s["q"])
    s["q"][..., 5] = 2.0**e * (torch.arange(6) % 3 - 1)
    s["k_cache"][..., 5] = 2.0**e * torch.randint(-1, 2, s["k_cache"].shape[:-1], generator=g)
    check_attend(cuda, s)
    check_attend(cuda, s, window=77)


def test_attend_to_nothing(cuda):
    s = attend_inputs(70, 2, 1, 16, 16, 16, 20, dtype=torch.float32)
    s["lengths"] = torch.zeros(70, dtype=torch.int64)
    for M in (20, 3):
        s["pages"] = s["pages"][:, :M]
        check_attend(cuda, s)


@pytest.mark.parametrize("window", [None, 5, 70])
@pytest.mark.parametrize("P", [4, 7, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_attend_places_without_a_part(cuda, window, P, dtype):
    s = attend_inputs(5, 4, 2, 80, 48, P, -(-200 // P), dtype=dtype)
    s["lengths"] = torch.tensor([0, 1, 130, 199, 200])
    poison(s, window)
    check_attend(cuda, s, window=window)


def test_attend_bad_pages_and_lengths(cuda):
    s = attend_inputs(6, 4, 2, 64, 64, 16, 20, dtype=torch.bfloat16)
    s["lengths"] = torch.tensor([300, 300, 300, 321, -7, 320])
    s["pages"][0, 3], s["pages"][1, 18] = -1, s["k_cache"].shape[0]
    s["pages"][2, 0] = 2**40
    check_attend(cuda, s)
    for kind in (torch.int32, torch.int64):
        d = to(s, cuda)
        d["pages"], d["lengths"] = d["pages"].clamp(max=2**31 - 1).to(kind), d["lengths"].int()
        check_attend(cuda, s, dev=d)


def test_attend_scale_and_large_scores(cuda):
    s = attend_inputs(3, 4, 2, 64, 64, 16, 20, dtype=torch.float32)
    s["q"] *= 100
    s["lengths"] = torch.tensor([1, 150, 320])
    want = attend_plain(**s, scale=3.0)
    got = paged_attention_step(**to(s, cuda), scale=3.0)
    # Scores of up to 1e4: 16 * 2^-24 of them is 1e-2 in a weight's logarithm.
    assert bool(torch.isfinite(got).all()) and off(got, want) <= 2e-2


def test_attend_infinite_scores(cuda):
    """A key that puts one score at -inf leaves it out; a NaN key is seen."""
    s = attend_inputs(2, 1, 1, 64, 64, 16, 4, dtype=torch.float32)
    s["lengths"] = torch.tensor([40, 40])
    s["q"] = s["q"].abs()
    s["k_cache"][s["pages"][0, 1], 0, 3] = -math.inf
    s["k_cache"][s["pages"][1, 2], 0, 2] = math.nan
    check_attend(cuda, s)


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_strides(cuda, dtype):
    s = attend_inputs(4, 6, 2, 64, 48, 16, 20, dtype=dtype)
    dev = to(s, cuda)
    for n in ("k_cache", "v_cache"):
        dev[n] = dev[n].transpose(1, 2).contiguous().transpose(1, 2)
    dev["q"] = torch.stack([dev["q"]] * 2, 2)[:, :, 0]
    dev["pages"] = torch.stack([dev["pages"]] * 2, -1)[..., 0]
    check_attend(cuda, s, dev=dev)
    both = torch.cat([dev["k_cache"], dev["v_cache"]], -1)  # keys and values side by side
    dev["k_cache"], dev["v_cache"] = both.split((64, 48), -1)
    check_attend(cuda, s, dev=dev)


def test_attend_queries_of_a_joined_projection(cuda):
    s = attend_inputs(4, 6, 2, 64, 64, 16, 20, dtype=torch.bfloat16)
    for pad in (0, 1, 4, 8):  # aligned or not
        dev = to(s, cuda)
        joined = torch.cat([dev["q"].flatten(1), dev["q"].flatten(1)[:, : 64 + pad]], 1)
        dev["q"] = joined[:, : 6 * 64].unflatten(1, (6, 64))
        check_attend(cuda, s, dev=dev)


def test_attend_unaligned(cuda):
    s = attend_inputs(4, 6, 2, 64, 64, 16, 20, dtype=torch.bfloat16)
    dev = to(s, cuda)
    for n in ("q", "k_cache", "v_cache"):
        t = torch.empty(dev[n].numel() + 1, dtype=torch.bfloat16, device=cuda)[1:]
        dev[n] = t.view(dev[n].shape).copy_(dev[n])
    check_attend(cuda, s, dev=dev)


def test_attend_repeats_bitwise(cuda):
    s = to(attend_inputs(20, 8, 2, 128, 128, 16, 100, dtype=torch.bfloat16), cuda)
    want = paged_attention_step(**s)
    for _ in range(5):
        assert torch.equal(paged_attention_step(**s), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16])
def test_offsets_past_32_bits(cuda, dtype):
    """Places beyond 2^32 bytes and 2^31 elements of a cache."""
    N, Hk, P, d = 270000, 1, 64, 128  # 2.2e9 elements
    k = torch.zeros(N, Hk, P, d, dtype=dtype, device=cuda)
    v = torch.zeros(N, Hk, P, d, dtype=dtype, device=cuda)
    g = torch.Generator().manual_seed(0)
    pages = torch.tensor([[N - 1, 5, N - 2], [N - 3, 262144, 7]])
    new = [torch.randn(2, 150, 1, d, generator=g).to(dtype) for _ in range(2)]
    q = torch.randn(2, 3, d, generator=g).to(dtype)
    paged_cache_append(new[0].to(cuda), new[1].to(cuda), k, v, pages.to(cuda),
                       torch.zeros(2, dtype=torch.int64, device=cuda))
    lengths = torch.tensor([150, 149])
    got = paged_attention_step(q.to(cuda), k, v, pages.to(cuda), lengths.to(cuda))
    small = pages.clone().flatten().argsort().argsort().view(2, 3)
    kc, vc = torch.zeros(6, 1, P, d), torch.zeros(6, 1, P, d)
    _, kc, vc = append_plain(new[0], new[1], kc, vc, small, torch.zeros(2))
    assert off(got, attend_plain(q, kc, vc, small, lengths)) <= ATTEND[dtype]
    for b in range(2):
        assert torch.equal(k[pages[b, 0], 0].cpu().double(), new[0][b, :64, 0].double())
    assert int((k != 0).any(-1).sum()) == 300


def test_on_another_stream(cuda):
    s = attend_inputs(20, 8, 2, 128, 128, 16, 100, dtype=torch.bfloat16)
    want = paged_attention_step(**to(s, cuda))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        dev = to(s, cuda)
        got = [paged_attention_step(**dev) for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(t, want) for t in got)


def test_in_graphs(cuda):
    """Two captured steps, of growing sequences, replayed in turn with eager calls between."""
    B, H, Hk, d, P, M = 3, 8, 2, 64, 16, 8
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(cuda)  # noqa: E731
    kc, vc = r(B * M, Hk, P, d), r(B * M, Hk, P, d)
    kc2, vc2 = kc.clone(), vc.clone()
    pages = tables(B, M, B * M, g).to(cuda)
    start = torch.tensor([0, 20, 100], device=cuda)
    at = start.clone()
    f = (100.0 ** -torch.linspace(0, 1, d // 2)).to(cuda)
    k, v, q = r(B, 1, Hk, d), r(B, 1, Hk, d), r(B, 1, H, d)

    def step(kc, vc, at):
        turn = paged_cache_append(k, v, kc, vc, pages, at, q=q, frequencies=f)
        return paged_attention_step(turn[:, 0], kc, vc, pages, at + 1)

    graphs = []
    for _ in range(2):
        step(kc2.clone(), vc2.clone(), at)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = step(kc, vc, at)
        graphs.append((graph, o))
    for i in range(6):
        for t in (k, v, q):
            t.copy_(r(*t.shape))
        at.copy_(start + i)
        graph, o = graphs[i % 2]
        graph.replay()
        want = step(kc2, vc2, at)
        torch.cuda.synchronize()
        assert torch.equal(o, want), i
        assert torch.equal(kc, kc2) and torch.equal(vc, vc2), i


def test_attend_declines(cuda):
    s = attend_inputs(3, 4, 2, 64, 64, 16, 20)
    with pytest.raises(RuntimeError, match="float64"):
        paged_attention_step(**to(s, cuda))
    s = attend_inputs(3, 4, 2, 257, 64, 16, 20, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="256"):
        paged_attention_step(**to(s, cuda))
