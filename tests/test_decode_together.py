"""A beam search over a paged cache as a decoder runs it: prompts appended and attended to, one
token a step after that, beams that share pages of one token and follow their parents by their page
tables.  Against a decoder that keeps nothing and attends over each beam's whole text again."""

import pytest
import torch

from mingru_amd import beam_select, paged_attention_step, paged_cache_append, reorder_states

B, K, H, HK, D, V, END = 3, 4, 4, 2, 16, 23, 5
STEPS = 7


def weights(dtype, device):
    g = torch.Generator().manual_seed(0)
    r = lambda *s, std: (torch.randn(*s, generator=g, dtype=torch.float64) * std).to(device, dtype)  # noqa: E731
    w = dict(embed=r(V, 32, std=1.0), q=r(32, H * D, std=0.4), k=r(32, HK * D, std=0.4),
             v=r(32, HK * D, std=0.4), o=r(H * D, 32, std=0.3), head=r(32, V, std=0.8))
    w["f"] = (100.0 ** -(torch.arange(D // 2, dtype=torch.float64) / (D // 2))).to(device)
    return w


def project(w, x):
    return [(x @ w[n]).unflatten(-1, (-1, D)) for n in "qkv"]


def logits_of(w, x, o):
    return (x + o.flatten(-2) @ w["o"]) @ w["head"]


def whole(w, tokens):
    """Logits after one text, everything formed anew."""
    x = w["embed"][tokens]
    q, k, v = project(w, x)
    n = torch.arange(len(tokens), dtype=torch.float64)

    def turn(t):
        c, s = (f(n[:, None] * w["f"])[:, None] for f in (torch.cos, torch.sin))
        a, b = t[..., : D // 2], t[..., D // 2 :]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k = turn(q)[-1], turn(k).repeat_interleave(H // HK, 1)
    p = torch.softmax((q * k).sum(-1) * D**-0.5, 0)
    return logits_of(w, x[-1], (p[..., None] * v.repeat_interleave(H // HK, 1)).sum(0))


def search_whole(prompts, lengths):
    w = weights(torch.float64, "cpu")
    out = []
    for row, n in zip(prompts, lengths):
        beams = [(0.0, row[:n].tolist(), False)]
        for _ in range(STEPS):
            every = []
            for k, (score, text, over) in enumerate(beams):
                if over:
                    every.append((-score, k, END, True))
                    continue
                logp = torch.log_softmax(whole(w, torch.tensor(text)), 0)
                every += [(-(score + float(logp[t])), k, t, t == END) for t in range(V)]
            beams = [(-c, beams[k][1] + [t], over) for c, k, t, over in sorted(every)[:K]]
        out.append(beams)
    return out


def search_paged(prompts, lengths, dtype, device):
    """Scores (B, K) and texts (B, K, STEPS)."""
    w = weights(dtype, device)
    prompts, lengths = prompts.to(device), lengths.to(device)
    T = prompts.shape[1]
    M = T + STEPS
    kc = torch.full((B * T + STEPS * B * K, HK, 1, D), float("nan"), dtype=dtype, device=device)
    vc = kc.clone()
    pages = torch.full((B, M), -1, dtype=torch.int32, device=device)
    pages[:, :T] = torch.arange(B * T, device=device).view(B, T)
    # The prompts: all keys and values at once, then the last token's attention.
    x = w["embed"][prompts]
    q, k, v = project(w, x)
    q = paged_cache_append(k, v, kc, vc, pages, torch.zeros(B, dtype=torch.int64, device=device), q=q,
                           lengths=lengths, frequencies=w["f"])
    rows = torch.arange(B, device=device)
    o = paged_attention_step(q[rows, lengths - 1], kc, vc, pages, lengths)
    x, scores, finished = x[rows, lengths - 1], torch.zeros(B, 1, device=device, dtype=torch.promote_types(dtype, torch.float32)), None
    at, texts = lengths, torch.zeros(B, 0, STEPS, dtype=torch.int64, device=device)
    texts = torch.zeros(B, STEPS, dtype=torch.int64, device=device)
    for step in range(STEPS):
        logits = logits_of(w, x, o).view(B, -1, V)
        scores, parent, token, finished = beam_select(logits, scores, K, end=END, finished=finished)
        pages, at, texts = reorder_states((pages, at, texts), parent)
        texts[:, step] = token.flatten()
        if step + 1 == STEPS:
            break
        # A new page for each beam: those before are shared, and written no more.
        new = B * T + step * B * K + torch.arange(B * K, device=device)
        pages.scatter_(1, at[:, None], new[:, None].to(pages.dtype))
        x = w["embed"][token.flatten()]
        q, k, v = project(w, x[:, None])
        q = paged_cache_append(k, v, kc, vc, pages, at, q=q, frequencies=w["f"])
        at = at + 1
        o = paged_attention_step(q[:, 0], kc, vc, pages, at)
    return scores, texts.view(B, K, STEPS)


def check(dtype, device, tol):
    g = torch.Generator().manual_seed(1)
    prompts, lengths = torch.randint(0, V, (B, 9), generator=g), torch.tensor([9, 1, 6])
    scores, texts = search_paged(prompts, lengths, dtype, device)
    for b, beams in enumerate(search_whole(prompts, lengths.tolist())):
        assert texts[b].tolist() == [text[int(lengths[b]):] for _, text, _ in beams], b
        for a, (c, _, _) in zip(scores[b].tolist(), beams):
            assert abs(a - c) <= tol * max(1.0, abs(c))


def test_search_over_pages():
    check(torch.float64, "cpu", 1e-10)


@pytest.mark.gpu
def test_gpu_search_over_pages(cuda, monkeypatch):
    # Seven steps of logits of about 10, each a sum of 64 products of sums of 32, in 32 bits: far
    # less than 1e-4 together; no two candidates at a border are that close.
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    check(torch.float32, cuda, 1e-4)
