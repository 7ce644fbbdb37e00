"""``paged_cache_append`` and ``paged_attention_step`` in their eager bodies: against the
definition token by token in float64, left-out tokens, masked places, and refusals."""

import math

import pytest
import torch

from mingru_amd import paged_attention_step, paged_cache_append


def turned(x, position, frequencies, interleaved):
    """One head's row (d) of float64, rotated."""
    x = x.clone()
    n = len(frequencies)
    for i, f in enumerate(frequencies.tolist()):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        c, s = math.cos(position * f), math.sin(position * f)
        x[a], x[b] = float(x[a] * c - x[b] * s), float(x[b] * c + x[a] * s)
    return x


def append_plain(k, v, k_cache, v_cache, pages, start, q=None, lengths=None, frequencies=None,
                 interleaved=False):
    """New caches and queries in float64; places that a token must not go to are left out."""
    k, v, k_cache, v_cache = (t.detach().double().cpu().clone() for t in (k, v, k_cache, v_cache))
    q = None if q is None else q.detach().double().cpu().clone()
    frequencies = torch.zeros(0) if frequencies is None else frequencies.detach().double().cpu()
    B, T, Hk, _ = k.shape
    N, _, P, _ = k_cache.shape
    for b in range(B):
        n = T if lengths is None else min(T, max(0, int(lengths[b])))
        if q is not None:
            q[b, n:] = 0
        for t in range(n):
            at = int(start[b]) + t
            lost = not 0 <= at < pages.shape[1] * P or int(pages[b, at // P]) >= N
            for h in range(0 if q is None else q.shape[2]):
                q[b, t, h] = turned(q[b, t, h], at, frequencies, interleaved)
                if lost:
                    q[b, t, h] = math.nan
            if lost or int(pages[b, at // P]) < 0:
                continue
            for h in range(Hk):
                k_cache[int(pages[b, at // P]), h, at % P] = turned(k[b, t, h], at, frequencies,
                                                                    interleaved)
                v_cache[int(pages[b, at // P]), h, at % P] = v[b, t, h]
    return q, k_cache, v_cache


def attend_plain(q, k_cache, v_cache, pages, lengths, scale=None, window=None):
    """(B, H, dv) in float64."""
    q, k_cache, v_cache = (t.detach().double().cpu() for t in (q, k_cache, v_cache))
    B, H, dk = q.shape
    N, Hk, P, dv = v_cache.shape
    scale = dk**-0.5 if scale is None else scale
    out = torch.zeros(B, H, dv, dtype=torch.float64)
    for b in range(B):
        n = max(0, int(lengths[b]))
        rows = range(max(0, n - window) if window else 0, n)
        if n > pages.shape[1] * P or any(not 0 <= int(pages[b, j // P]) < N for j in rows):
            out[b] = math.nan
            continue
        if n == 0:
            continue
        page, slot = (torch.tensor([f(j) for j in rows])
                      for f in (lambda j: int(pages[b, j // P]), lambda j: j % P))
        for h in range(H):
            k, v = (c[page, h // (H // Hk), slot] for c in (k_cache, v_cache))
            out[b, h] = torch.softmax(scale * (k @ q[b, h]), 0) @ v
    return out


def tables(B, M, N, g):
    """Distinct pages of N in no order."""
    assert B * M <= N
    return torch.randperm(N, generator=g)[: B * M].view(B, M)


def append_inputs(B, T, H, Hk, dk, dv, P, M, n, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
    N = B * M + 3
    return dict(k=r(B, T, Hk, dk), v=r(B, T, Hk, dv), k_cache=r(N, Hk, P, dk),
                v_cache=r(N, Hk, P, dv), pages=tables(B, M, N, g),
                start=torch.randint(0, M * P - T + 1, (B,), generator=g),
                q=r(B, T, H, dk) if H else None,
                frequencies=100.0 ** -torch.linspace(0, 1, n, dtype=torch.float64) if n else None)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n", [0, 1, 3, 4])
@pytest.mark.parametrize("ragged", [False, True])
def test_append(interleaved, n, ragged):
    s = append_inputs(3, 5, 4, 2, 8, 6, 3, 4, n)
    if ragged:
        s["lengths"] = torch.tensor([5, 0, 2])
    want = append_plain(**s, interleaved=interleaved)
    got = paged_cache_append(**s, interleaved=interleaved)
    for a, b in zip((got, s["k_cache"], s["v_cache"]), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_far_positions_turn_by_64_bit_angles():
    s = append_inputs(1, 1, 1, 1, 2, 1, 1, 1, 1, dtype=torch.float32)
    far = 2**30 + 1
    s["pages"] = torch.zeros(1, 1, dtype=torch.int64).expand(1, far + 1)
    s["start"] = torch.tensor([far])
    want, *_ = append_plain(**s)
    assert torch.allclose(paged_cache_append(**s).double(), want, rtol=0, atol=1e-6)


def test_negative_pages_are_not_kept():
    s = append_inputs(2, 4, 2, 1, 4, 4, 2, 4, 2)
    s["start"] = torch.tensor([0, 2])
    s["pages"][0, 1] = -1
    want = append_plain(**s)
    got = paged_cache_append(**s)
    for a, b in zip((got, s["k_cache"], s["v_cache"]), want):
        assert torch.allclose(a, b)


def test_padding_is_not_read():
    s = append_inputs(2, 3, 2, 1, 4, 4, 2, 4, 2)
    s["lengths"] = torch.tensor([1, 0])
    for n in "qkv":
        s[n][0, 1:] = math.nan
        s[n][1] = math.inf
    s["start"][1] = 10**6  # of no token
    want = append_plain(**s)
    got = paged_cache_append(**s)
    assert torch.isfinite(got).all()
    for a, b in zip((got, s["k_cache"], s["v_cache"]), want):
        assert torch.allclose(a, b)


def test_append_of_nothing():
    s = append_inputs(2, 0, 2, 1, 4, 4, 2, 2, 2)
    before = s["k_cache"].clone()
    assert paged_cache_append(**s).shape == (2, 0, 2, 4)
    assert torch.equal(s["k_cache"], before)
    s["q"] = None
    assert paged_cache_append(**s) is None


@pytest.mark.parametrize("change, error", [
    (dict(start=torch.tensor([100, 0])), IndexError),
    (dict(start=torch.tensor([0, -1])), IndexError),
    (dict(pages=torch.full((2, 4), 99)), IndexError),
    (dict(pages=torch.zeros(3, 4, dtype=torch.int64)), ValueError),
    (dict(pages=torch.zeros(2, 4)), TypeError),
    (dict(start=torch.zeros(2)), TypeError),
    (dict(start=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(lengths=torch.ones(2, dtype=torch.bool)), TypeError),
    (dict(k=torch.zeros(2, 4, 1, 5, dtype=torch.float64)), ValueError),
    (dict(k=torch.zeros(2, 4, 1, 4)), TypeError),
    (dict(v=torch.zeros(2, 4, 1, 5, dtype=torch.float64)), ValueError),
    (dict(q=torch.zeros(2, 4, 2, 5, dtype=torch.float64)), ValueError),
    (dict(q=torch.zeros(2, 4, 2, 4)), TypeError),
    (dict(frequencies=torch.zeros(3)), ValueError),
    (dict(frequencies=torch.zeros(0)), ValueError),
    (dict(frequencies=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(k_cache=torch.zeros(1, 1, 2, 4, dtype=torch.float64).expand(11, 1, 2, 4)), ValueError),
    (dict(k_cache=torch.zeros(11, 1, 0, 4, dtype=torch.float64)), ValueError),
])
def test_append_refuses(change, error):
    s = append_inputs(2, 4, 2, 1, 4, 4, 2, 4, 2)
    before = s["v_cache"].clone()
    with pytest.raises(error):
        paged_cache_append(**{**s, **change})
    assert torch.equal(s["v_cache"], before)


def attend_inputs(B, H, Hk, dk, dv, P, M, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
    N = B * M + 3
    return dict(q=r(B, H, dk), k_cache=r(N, Hk, P, dk), v_cache=r(N, Hk, P, dv),
                pages=tables(B, M, N, g), lengths=torch.randint(0, M * P + 1, (B,), generator=g))


@pytest.mark.parametrize("window", [None, 1, 4, 1000])
@pytest.mark.parametrize("H, Hk", [(1, 1), (4, 4), (6, 2)])
def test_attend(window, H, Hk):
    s = attend_inputs(5, H, Hk, 8, 6, 3, 7)
    s["lengths"][:3] = torch.tensor([0, 1, 21])
    want = attend_plain(**s, window=window)
    got = paged_attention_step(**s, window=window)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)
    assert torch.equal(got[0], torch.zeros_like(got[0]))
    assert torch.allclose(paged_attention_step(**s, scale=0.5, window=window),
                          attend_plain(**s, scale=0.5, window=window), rtol=1e-12, atol=1e-12)


def poison(s, window):
    """NaN and infinities in every place that has no part in the result."""
    P = s["k_cache"].shape[2]
    used = torch.zeros(s["k_cache"].shape[0], P, dtype=torch.bool)
    for b, n in enumerate(s["lengths"].tolist()):
        for j in range(max(0, n - window) if window else 0, n):
            used[s["pages"][b, j // P], j % P] = True
        first = (max(0, n - window) if window else 0) // P
        last = -(-n // P)
        s["pages"][b, :first], s["pages"][b, last:] = -1, 10**6
    for name in ("k_cache", "v_cache"):
        c = s[name].transpose(1, 2)
        c[~used] = math.nan if name == "k_cache" else math.inf


@pytest.mark.parametrize("window", [None, 5])
def test_places_without_a_part_do_not_matter(window):
    s = attend_inputs(4, 4, 2, 8, 6, 4, 6)
    s["lengths"] = torch.tensor([0, 1, 13, 24])
    want = attend_plain(**s, window=window)
    poison(s, window)
    got = paged_attention_step(**s, window=window)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-12)


def test_other_orders_of_the_cache():
    s = attend_inputs(3, 4, 2, 8, 6, 4, 6)
    want = attend_plain(**s)
    for n in ("k_cache", "v_cache"):
        s[n] = s[n].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.allclose(paged_attention_step(**s), want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("change, error", [
    (dict(lengths=torch.tensor([99, 0])), IndexError),
    (dict(pages=torch.full((2, 6), -1)), IndexError),
    (dict(pages=torch.full((2, 6), 15)), IndexError),
    (dict(lengths=torch.tensor([1.0, 2.0])), TypeError),
    (dict(lengths=torch.tensor([1])), ValueError),
    (dict(pages=torch.zeros(6, dtype=torch.int64)), ValueError),
    (dict(q=torch.zeros(2, 3, 8, dtype=torch.float64)), ValueError),
    (dict(q=torch.zeros(2, 4, 7, dtype=torch.float64)), ValueError),
    (dict(q=torch.zeros(2, 4, 8)), TypeError),
    (dict(q=torch.zeros(2, 1, 4, 8, dtype=torch.float64)), ValueError),
    (dict(v_cache=torch.zeros(15, 2, 5, 6, dtype=torch.float64)), ValueError),
    (dict(window=0), ValueError),
    (dict(window=2.5), ValueError),
    (dict(window=True), ValueError),
])
def test_attend_refuses(change, error):
    s = attend_inputs(2, 4, 2, 8, 6, 4, 6)
    s["lengths"] = torch.tensor([5, 24])
    with pytest.raises(error):
        paged_attention_step(**{**s, **change})


def test_no_sequences():
    s = attend_inputs(2, 4, 2, 8, 6, 4, 6)
    for n in ("q", "pages", "lengths"):
        s[n] = s[n][:0]
    assert paged_attention_step(**s).shape == (0, 4, 6)


def test_appended_tokens_are_attended_to():
    """A prompt, then tokens one by one, against attention over everything at once."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    B, H, Hk, d, P, M, T = 2, 4, 2, 8, 3, 4, 10
    k, v, q = r(B, T, Hk, d), r(B, T, Hk, d), r(B, T, H, d)
    f = 100.0 ** -torch.linspace(0, 1, 4, dtype=torch.float64)
    kc, vc = r(B * M, Hk, P, d), r(B * M, Hk, P, d)
    pages = tables(B, M, B * M, g)
    prompt = torch.tensor([4, 6])
    pad = [torch.cat([t[:, :6]], 1) for t in (k, v, q)]
    paged_cache_append(pad[0], pad[1], kc, vc, pages, torch.zeros(2, dtype=torch.int64), q=pad[2],
                       lengths=prompt, frequencies=f)
    for step in range(4):
        at = prompt + step
        new = [t[torch.arange(B), at][:, None] for t in (k, v, q)]
        turn = paged_cache_append(new[0], new[1], kc, vc, pages, at, q=new[2], frequencies=f)
        o = paged_attention_step(turn[:, 0], kc, vc, pages, at + 1)
        for b in range(B):
            n = int(at[b]) + 1
            for h in range(H):
                kk = torch.stack([turned(k[b, j, h // 2], j, f, False) for j in range(n)])
                w = torch.softmax(kk @ turned(q[b, n - 1, h], n - 1, f, False) * d**-0.5, 0)
                assert torch.allclose(o[b, h], w @ v[b, :n, h // 2], rtol=1e-10, atol=1e-10)
