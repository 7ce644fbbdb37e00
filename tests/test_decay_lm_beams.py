"""Beam search of the example model: as wide as all continuations it finds the likeliest one, a
beam alone is the greedy choice, and what has ended stays ended; on the GPU the kernels give the
CPU's tokens."""

import itertools

import pytest
import torch

from mingru_amd.decay_lm import DecayLM


def model(vocabulary=6, seed=0):
    torch.manual_seed(seed)
    m = DecayLM(vocabulary, d_model=32, n_layers=2, n_heads=2)
    with torch.no_grad():
        m.head.weight.mul_(8.0)  # far from even odds
    return m


def score(m, prompt, more, end=None):
    """Log probability of tokens after one prompt, up to the first ``end``."""
    y, _ = m(torch.cat([prompt, torch.tensor(more)])[None])
    logp = torch.log_softmax(m.head(y), -1)[0, len(prompt) - 1 :].detach()
    total = 0.0
    for i, t in enumerate(more):
        total += float(logp[i, t])
        if t == end:
            break
    return total


@pytest.mark.parametrize("end", [None, 2])
def test_all_continuations(end):
    m = model().double()
    g = torch.Generator().manual_seed(1)
    prompts = torch.randint(0, 6, (3, 5), generator=g)
    got = m.generate(prompts, 3, beams=216, end=end)
    for prompt, tokens in zip(prompts, got.tolist()):
        best = max((c for c in itertools.product(range(6), repeat=3)
                    if end is None or all(b == end for a, b in zip(c, c[1:]) if a == end)),
                   key=lambda c: score(m, prompt, c, end))
        assert tokens == list(best)


def test_one_beam_is_greedy():
    m = model().double()
    prompts = torch.randint(0, 6, (3, 5), generator=torch.Generator().manual_seed(2))
    assert torch.equal(m.generate(prompts, 6, beams=1, end=5)[:, :1], m.generate(prompts, 1))
    y, state = m(prompts)
    assert torch.equal(m._search(y[:, -1], state, 6, 1, None), m.generate(prompts, 6))


def test_padded_prompts_search_as_their_own():
    m = model().double()
    tokens = torch.randint(0, 6, (3, 8), generator=torch.Generator().manual_seed(3))
    lengths = torch.tensor([8, 3, 1])
    got = m.generate(tokens, 5, lengths, beams=4)
    for row, n in enumerate(lengths.tolist()):
        assert torch.equal(got[row : row + 1], m.generate(tokens[row : row + 1, :n], 5, beams=4))


def test_refusals():
    with pytest.raises(ValueError, match="beams"):
        model().generate(torch.zeros(1, 2, dtype=torch.int64), 3, beams=0)
    with pytest.raises(ValueError, match="end"):
        model().generate(torch.zeros(1, 2, dtype=torch.int64), 3, beams=2, end=6)


@pytest.mark.gpu
@pytest.mark.parametrize("end", [None, 3])
def test_gpu_gives_the_cpu_tokens(cuda, monkeypatch, end):
    m = model(50)
    prompts = torch.randint(0, 50, (5, 40), generator=torch.Generator().manual_seed(4))
    lengths = torch.tensor([40, 1, 17, 39, 8])
    want = model(50).double().generate(prompts, 12, lengths, beams=4, end=end)
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    got = m.to(cuda).generate(prompts.to(cuda), 12, lengths.to(cuda), beams=4, end=end)
    assert torch.equal(got.cpu(), want)
