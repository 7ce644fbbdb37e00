"""``beam_select`` and ``reorder_states`` in their eager bodies: against every candidate ranked in
float64, ties, beams without a candidate, and refusals."""

import collections
import math

import pytest
import torch

from mingru_amd import beam_select, reorder_states


def beam_plain(logits, scores, width=None, *, end=None, finished=None):
    """Lists of (score, parent, token) for each search, from the definition."""
    B, K, V = logits.shape
    out = []
    for b in range(B):
        all_ = []
        for k in range(K):
            x = [float(t) for t in logits[b, k]]
            s = float(scores[b, k])
            over = finished is not None and bool(finished[b, k])
            top = max((t for t in x if not math.isnan(t)), default=-math.inf)
            total = math.nan
            if all(not math.isnan(t) and t != math.inf for t in x) and top > -math.inf:
                total = top + math.log(math.fsum(math.exp(t - top) for t in x))
            for v in range(V):
                if not math.isfinite(s):
                    c = -math.inf
                elif over:
                    c = s if v == end else -math.inf
                else:
                    c = s + (x[v] - total) if math.isfinite(total) else -math.inf
                all_.append((-c, k, v))
        all_.sort()
        out.append([(-c, k, v) for c, k, v in all_[: K if width is None else width]])
    return out


def check_beam(got, want, end=None, finished=None, tol=1e-12):
    score, parent, token = (t.cpu() for t in got[:3])
    for b, rows in enumerate(want):
        assert parent[b].tolist() == [k for _, k, _ in rows], b
        assert token[b].tolist() == [v for _, _, v in rows], b
        for a, (c, _, _) in zip(score[b].tolist(), rows):
            assert a == c or abs(a - c) <= tol * max(1.0, abs(c)), (b, a, c)
        if end is not None:
            assert got[3].cpu()[b].tolist() == [
                v == end or (finished is not None and bool(finished[b, k])) for _, k, v in rows]


def beam_inputs(B, K, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, K, V, generator=g, dtype=torch.float64) * 2,
            -10 * torch.rand(B, K, generator=g, dtype=torch.float64))


@pytest.mark.parametrize("B, K, V, width", [(1, 1, 7, 1), (2, 3, 11, None), (3, 4, 5, 20),
                                            (2, 2, 9, 6), (1, 5, 1, 5), (2, 1, 30, 4)])
def test_select(B, K, V, width):
    logits, scores = beam_inputs(B, K, V)
    got = beam_select(logits, scores, width)
    check_beam(got, beam_plain(logits, scores, width))
    assert got[0].dtype == torch.float64 and got[1].dtype == got[2].dtype == torch.int64


def test_ties_go_to_the_lower_beam_then_the_lower_token():
    logits = torch.zeros(1, 3, 4)
    got = beam_select(logits, torch.zeros(1, 3), 6)
    assert got[1].tolist() == [[0, 0, 0, 0, 1, 1]] and got[2].tolist() == [[0, 1, 2, 3, 0, 1]]
    logits[0, 1, 2], logits[0, 1, 1] = 0.0, -0.0
    got = beam_select(logits, torch.tensor([[-1.0, 0.0, -1.0]]), 3)
    assert got[2].tolist() == [[0, 1, 2]]
    assert got[0].dtype == torch.float32


@pytest.mark.parametrize("size", [1.0, 1e9, 3e37, 1e300])
def test_large_logits_keep_their_rows_weight(size):
    """Beams that differ only in how many tokens share a row."""
    logits = torch.full((1, 3, 8), -math.inf, dtype=torch.float64)
    logits[0, 0, :4], logits[0, 1, 5:7], logits[0, 2] = size, -size, size
    score, parent, token = beam_select(logits, torch.tensor([[0.0, -0.1, 0.0]]), 7)
    assert parent.tolist() == [[1, 1, 0, 0, 0, 0, 2]] and token.tolist() == [[5, 6, 0, 1, 2, 3, 0]]
    want = torch.tensor([-0.1 - math.log(2)] * 2 + [-math.log(4)] * 4 + [-math.log(8)])
    assert torch.allclose(score[0], want.double(), atol=1e-6)  # the scores are of 32 bits


def odd_beams(K=8, V=13, width=20, seed=1):
    """Beams that have ended, that have no finite score or sum, and masked tokens."""
    logits, scores = beam_inputs(1, K, V, seed)
    logits[0, 0, 3:] = -math.inf
    logits[0, 1] = -math.inf
    logits[0, 2, 5] = math.nan
    logits[0, 3, 6] = math.inf
    scores[0, 4], scores[0, 5] = -math.inf, math.nan
    finished = torch.zeros(1, K, dtype=torch.bool)
    finished[0, 4] = finished[0, 6] = True
    logits[0, 6] = math.nan  # not read
    return logits, scores, finished


@pytest.mark.parametrize("width", [1, 4, 20, 60])
@pytest.mark.parametrize("end", [0, 7, 12])
def test_beams_without_candidates(width, end):
    logits, scores, finished = odd_beams()
    got = beam_select(logits, scores, width, end=end, finished=finished)
    check_beam(got, beam_plain(logits, scores, width, end=end, finished=finished), end, finished)


def test_end_without_finished():
    logits, scores = beam_inputs(2, 3, 6)
    got = beam_select(logits, scores, 8, end=4)
    check_beam(got, beam_plain(logits, scores, 8), 4)


@pytest.mark.parametrize("kw, error", [
    (dict(width=0), ValueError), (dict(width=37), ValueError), (dict(width=2.5), ValueError),
    (dict(width=True), ValueError), (dict(end=6), ValueError), (dict(end=-1), ValueError),
    (dict(finished=torch.zeros(2, 3, dtype=torch.bool)), ValueError),
    (dict(end=1, finished=torch.zeros(2, 3)), TypeError),
    (dict(end=1, finished=torch.zeros(3, 2, dtype=torch.bool)), ValueError),
])
def test_select_refuses(kw, error):
    logits, scores = beam_inputs(2, 3, 6)
    with pytest.raises(error):
        beam_select(logits, scores, **kw)


def test_select_refuses_shapes():
    logits, scores = beam_inputs(2, 3, 6)
    for a, b in ((logits[0], scores), (logits, scores[:, :2]), (logits[..., :0], scores)):
        with pytest.raises(ValueError):
            beam_select(a, b)
    with pytest.raises(TypeError):
        beam_select(logits.long(), scores)
    assert [t.shape for t in beam_select(logits[:0], scores[:0], 4)] == [(0, 4)] * 3


Pair = collections.namedtuple("Pair", "a b")


def test_reorder():
    rows = torch.arange(6)
    states = [rows[:, None] * torch.ones(6, 3), None, {"x": rows.to(torch.bfloat16)},
              (rows[:, None, None].expand(6, 2, 2), Pair(rows % 2 == 0, torch.zeros(6, 0)))]
    parents = torch.tensor([[2, 0, 0, 1], [1, 1, 2, 0]])
    at = torch.tensor([2, 0, 0, 1, 4, 4, 5, 3])
    got = reorder_states(states, parents)
    assert torch.equal(got[0], states[0][at]) and got[1] is None
    assert got[2]["x"].dtype == torch.bfloat16 and torch.equal(got[2]["x"], states[2]["x"][at])
    assert isinstance(got[3], tuple) and torch.equal(got[3][0], states[3][0][at])
    assert isinstance(got[3][1], Pair) and torch.equal(got[3][1].a, states[3][1].a[at])
    assert got[3][1].b.shape == (8, 0)
    assert torch.equal(reorder_states(states[0], parents.int()), states[0][at])
    assert reorder_states([None], parents) == [None]


def test_reorder_spreads_a_prompt_over_beams():
    x = torch.randn(3, 4)
    got = reorder_states(x, torch.zeros(3, 5, dtype=torch.int64))
    assert torch.equal(got, x.repeat_interleave(5, 0))


@pytest.mark.parametrize("states, parents, error", [
    (torch.zeros(6, 2), torch.tensor([[0, 3], [0, 0]]), IndexError),
    (torch.zeros(6, 2), torch.tensor([[0, -1], [0, 0]]), IndexError),
    (torch.zeros(5, 2), torch.tensor([[0], [0]]), ValueError),
    ([torch.zeros(6, 2), torch.zeros(4, 2)], torch.tensor([[0], [0]]), ValueError),
    (torch.zeros(()), torch.tensor([[0]]), ValueError),
    (torch.zeros(6, 2), torch.tensor([0, 0]), ValueError),
    (torch.zeros(6, 2), torch.zeros(2, 2), TypeError),
    ([torch.zeros(6, 2), 3], torch.tensor([[0], [0]]), TypeError),
    (torch.zeros(6, 2), [[0], [0]], TypeError),
])
def test_reorder_refuses(states, parents, error):
    with pytest.raises(error):
        reorder_states(states, parents)
