"""``beam_select`` and ``reorder_states`` kernels against every candidate ranked in float64.

Scores: fp32 exponentials (2^-22 off at most where they count) summed in fp32 over a lane's part
of a row (at most 2^-16 of it, in disorder far less), the rest in fp64, and one rounding of the
result: 1e-6 of it, with the logarithms here no larger than the scores.  Parents and tokens are
equal: no two candidates' scores of one test are that close without being equal.
"""

import math

import pytest
import torch

from mingru_amd import beam_select, reorder_states
from tests.test_beam_search import beam_inputs, beam_plain, check_beam, odd_beams

pytestmark = pytest.mark.gpu
TOL = 1e-6


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def exact(logits, scores, width, end=None, finished=None):
    """The eager body in float64, on the CPU."""
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MINGRU_SCAN", "eager")
        return beam_select(logits.cpu().double(), scores.cpu().double(), width, end=end,
                           finished=None if finished is None else finished.cpu())


def check_near(logits, scores, width):
    """As ``check`` where scores of two beams may be nearer than the roundings of their rows' sums,
    2^-24 of each or more: such candidates may change places.  Each is then a candidate of its own,
    with its own score, which is also that of its place."""
    want = exact(logits, scores, width)
    score, parent, token = (t.cpu() for t in beam_select(logits, scores, width))
    x = torch.log_softmax(logits.cpu().double(), -1) + scores.cpu().double()[..., None]
    own = x.flatten(1).gather(1, parent * logits.shape[2] + token)
    for other in (own, want[0]):
        assert not bool(((score.double() - other).abs() > TOL * other.abs().clamp(min=1.0)).any())
    assert not bool((score[:, 1:] > score[:, :-1]).any())
    assert all(len(set(zip(p, t))) == width for p, t in zip(parent.tolist(), token.tolist()))


def check(logits, scores, width, end=None, finished=None):
    want = exact(logits, scores, width, end, finished)
    got = beam_select(logits, scores, width, end=end, finished=finished)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int64
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    a, b = got[0].double().cpu(), want[0]
    assert torch.equal(torch.isfinite(a), torch.isfinite(b))
    assert not bool(((a - b).abs() > TOL * b.abs().clamp(min=1.0)).any()), float((a - b).abs().max())
    if end is not None:
        assert torch.equal(got[3].cpu(), want[3])


def inputs(cuda, B, K, V, dtype, seed=0):
    logits, scores = beam_inputs(B, K, V, seed)
    return logits.to(dtype).to(cuda), scores.float().to(cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, K, V, width", [
    (1, 1, 1, 1), (1, 1, 5, 3), (2, 3, 11, 33), (3, 4, 2047, 4), (1, 4, 2048, 8), (2, 8, 2049, 64),
    (1, 2, 50257, 2), (1, 1, 131071, 64), (1, 1, 300007, 64), (40, 5, 1000, 5), (3, 64, 700, 64), (1, 256, 300, 40),
    (700, 1, 33, 7), (1, 1, 64, 64), (2, 2, 40, 64), (9, 16, 4096, 32)])
def test_sizes(cuda, dtype, B, K, V, width):
    check(*inputs(cuda, B, K, V, dtype), width)


@pytest.mark.parametrize("width", [1, 4, 20, 60])
@pytest.mark.parametrize("end", [0, 7, 12])
@pytest.mark.parametrize("V", [13, 5000])
def test_beams_without_candidates(cuda, width, end, V):
    logits, scores, finished = odd_beams(V=V)
    logits, scores = logits.float(), scores.float()
    if V == 13:
        check_beam([t.cpu() for t in beam_select(logits.to(cuda), scores.to(cuda), width, end=end,
                                                 finished=finished.to(cuda))],
                   beam_plain(logits, scores, width, end=end, finished=finished), end, finished,
                   tol=TOL)
    check(logits.to(cuda), scores.to(cuda), width, end, finished.to(cuda))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few", "masked", "lowest", "one"])
@pytest.mark.parametrize("V", [100, 9000])
def test_orders(cuda, dtype, kind, V):
    """Rows where every element, or none, beats the ones before, and rows full of ties."""
    g = torch.Generator().manual_seed(1)
    x = torch.zeros(2, 3, V)
    if kind == "rising":
        x += torch.arange(V) / 16
    elif kind == "falling":
        x -= torch.arange(V) / 16
    elif kind == "few":
        x += torch.randint(0, 3, (2, 3, V), generator=g)
    elif kind == "masked":
        x += torch.randn(2, 3, V, generator=g)
        x[..., torch.rand(V, generator=g) < 0.97] = -math.inf
    elif kind == "lowest":
        x += torch.finfo(dtype).min
        x[0, 0, 7] = 0.0
    elif kind == "one":
        x += -math.inf
        x[..., V - 1] = 3.0
    scores = -torch.rand(2, 3, generator=g)
    for width in (1, 6, 64):
        check(x.to(dtype).to(cuda), scores.to(cuda), width)


@pytest.mark.parametrize("kind", ["level", "ahead", "equal", "close", "finished", "dead", "spread"])
@pytest.mark.parametrize("B, K, V, width", [(1, 256, 3001, 64), (3, 64, 5000, 64), (2, 33, 9001, 50),
                                            (1, 200, 70, 64), (1, 256, 20011, 64)])
def test_many_beams(cuda, kind, B, K, V, width):
    """Candidates of one beam alone, of all, and far more of one score than are kept."""
    logits, scores = beam_inputs(B, K, V, 3)
    logits, scores, finished = logits.float(), scores.float(), None
    g = torch.Generator().manual_seed(5)
    if kind == "level":
        scores[:] = -1.0
    elif kind == "ahead":
        scores -= 100.0
        scores[:, K // 2] = -1.0
    elif kind == "equal":
        logits[:], scores[:] = 0.25, -2.0
    elif kind == "close":  # steps of a few roundings
        logits = torch.randint(0, 9, logits.shape, generator=g) * 2.0**-20
        scores[:] = -3.0
    elif kind == "finished":
        finished = torch.rand(B, K, generator=g) < 0.9
        scores -= 50.0 * torch.rand(B, K, generator=g)
    elif kind == "dead":  # fewer candidates than are kept
        logits[..., 3:] = -math.inf
        scores[:, 5:] = -math.inf
    elif kind == "spread":
        scores *= torch.logspace(-3, 9, K)
    end = None if finished is None else 11
    finished = None if finished is None else finished.to(cuda)
    if kind == "close":
        check_near(logits.to(cuda), scores.to(cuda), width)
    else:
        check(logits.to(cuda), scores.to(cuda), width, end, finished)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e4, 1e6, 1.2e6, 3e9, 1e20, 3e37, 3e38])
def test_large_logits(cuda, dtype, size):
    """Up to where a logit times log2 e leaves the type's range; equal ones share a row's weight."""
    g = torch.Generator().manual_seed(2)
    x = size * torch.randint(-1, 2, (2, 3, 5000), generator=g).float()
    x[0, 0] = size
    x[0, 1] = -size
    x[1, 2, 7:] = -size
    check(x.to(dtype).to(cuda), -torch.rand(2, 3, generator=g).to(cuda), 8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_start_anywhere(cuda, dtype):
    logits, scores = inputs(cuda, 3, 4, 3001, dtype)
    wide = torch.full((3, 4, 3040), math.nan, dtype=dtype, device=cuda)
    for at in (0, 1, 2, 3, 7, 8, 13, 39):
        wide[:] = math.nan
        wide[..., at : at + 3001] = logits
        check(wide[..., at : at + 3001], scores, 6)
    turned = logits.transpose(0, 1).contiguous().transpose(0, 1)
    check(turned, scores.t().contiguous().t(), 6)
    check(logits[:, ::2], scores[:, ::2], 6, 3, (torch.arange(12, device=cuda).view(3, 4) % 3 == 0)[:, ::2])
    check(logits.transpose(1, 2).contiguous().transpose(1, 2), scores, 6)


def test_score_types(cuda):
    logits, scores = inputs(cuda, 2, 4, 300, torch.float32)
    check(logits, scores.bfloat16(), 5)
    with pytest.raises(RuntimeError, match="32 bits"):
        beam_select(logits, scores.double())
    with pytest.raises(RuntimeError, match="float64"):
        beam_select(logits.double(), scores)
    with pytest.raises(RuntimeError, match="64"):
        beam_select(logits, scores, 65)
    with pytest.raises(RuntimeError, match="256"):
        beam_select(torch.zeros(1, 257, 3, device=cuda), torch.zeros(1, 257, device=cuda), 5)


def test_repeats_bitwise(cuda):
    logits, scores = inputs(cuda, 16, 8, 30000, torch.bfloat16)
    want = beam_select(logits, scores)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(beam_select(logits, scores), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.int32,
                                   torch.int64, torch.bool, torch.uint8, torch.float64,
                                   torch.complex64])
@pytest.mark.parametrize("shape", [(), (1,), (3,), (8, 5), (1024,), (1025,), (3, 1000), (0, 4),
                                   (17,), (4099,), (20001,)])
def test_reorder(cuda, dtype, shape):
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(6 * 4, *shape, generator=g) * 20).to(dtype).to(cuda)
    for W in (1, 4, 9):
        parents = torch.randint(0, 4, (6, W), generator=g)
        at = (parents + 4 * torch.arange(6)[:, None]).flatten().to(cuda)
        for kind in (torch.int64, torch.int32, torch.int8):
            got = reorder_states(x, parents.to(kind).to(cuda))
            assert got.dtype == x.dtype and torch.equal(got, x[at])


def test_reorder_many(cuda):
    """More tensors than a launch takes, of many sizes, strided and not, with None between."""
    g = torch.Generator().manual_seed(0)
    states = []
    for i in range(75):
        x = torch.randn(12, int(torch.randint(1, 3000, (), generator=g)), generator=g).to(cuda)
        if i % 5 == 1:
            x = x[:, ::2]
        if i % 5 == 2:
            x = torch.cat([x, x], 1)[:, 1 : x.shape[1] + 1]
        if i % 5 == 3:
            x = x.bfloat16()
        if i % 5 == 4:
            x = x[:1].expand(12, -1)
        states.append(None if i % 9 == 8 else x)
    parents = torch.randint(0, 4, (3, 5), generator=g)
    at = (parents + 4 * torch.arange(3)[:, None]).flatten().to(cuda)
    turned = torch.stack([parents.to(cuda)] * 2, 2).transpose(0, 1)[..., 0].t()
    for a, b in zip(reorder_states(states, turned), states):
        assert (a is None and b is None) or torch.equal(a, b[at])


def test_reorder_outside_parents_give_0(cuda):
    x = torch.randn(8, 100, device=cuda)
    got = reorder_states(x, torch.tensor([[0, 4], [-1, 3]], device=cuda))
    assert torch.equal(got[0], x[0]) and torch.equal(got[3], x[7])
    assert not bool(got[1].any()) and not bool(got[2].any())


def test_reorder_past_32_bits(cuda):
    x = torch.zeros(5, 2**30, dtype=torch.uint8, device=cuda)
    x[:, -3:] = torch.arange(15, device=cuda).view(5, 3).to(torch.uint8)
    got = reorder_states(x, torch.tensor([[4, 0, 3, 1, 2]], device=cuda))
    assert torch.equal(got[:, -3:], x[[4, 0, 3, 1, 2], -3:])
    assert int(got.sum(dtype=torch.int64)) == 105


def test_search_in_a_graph(cuda):
    """One step of a search, captured, replayed on new values with eager calls between."""
    logits, scores = inputs(cuda, 2, 4, 5000, torch.bfloat16)
    states = [torch.randn(8, 300, device=cuda), torch.randn(8, 7, device=cuda).bfloat16()]

    def step():
        score, parent, token, done = beam_select(logits, scores, end=3)
        return [score, parent, token, done, *reorder_states(states, parent)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(5):
        logits.copy_(beam_inputs(2, 4, 5000, i)[0])
        states[0].add_(1.0)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_on_another_stream(cuda):
    logits, scores = inputs(cuda, 16, 8, 30000, torch.float32)
    want = beam_select(logits, scores)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [beam_select(logits, scores) for _ in range(3)]
    stream.synchronize()
    assert all(torch.equal(a, b) for one in got for a, b in zip(one, want))


def test_reorder_resolves_views(cuda):
    """Conjugates and negatives that are only marked as such."""
    x = torch.randn(6, 5, dtype=torch.complex64, device=cuda)
    parents = torch.tensor([[2, 0], [1, 1]], device=cuda)
    at = torch.tensor([2, 0, 4, 4], device=cuda)
    for t in (x.conj(), x.conj().imag):
        assert torch.equal(reorder_states(t, parents), t.resolve_conj().resolve_neg()[at])
