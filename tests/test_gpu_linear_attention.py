"""``linear_attention`` kernels against the recurrence in float64: head sizes and lengths around
the tiles, shared keys, documents, padding, states in and out, strides, streams and graphs.

Tolerances, as the 2-norm of the difference over the 2-norm of the result.  fp32: three chained
products with sums of up to 128 terms of either sign, sqrt(128) 2^-24 each, and as much again
for the decays and the state's own sums: 6 * sqrt(128) * 2^-24 = 4e-6; the gradient of the
decays is a sum of terms that cancel, four times that.  bf16 outputs: the result and one operand
of its last product are rounded to 8 bits, 2 * 2^-8.  fp32 outputs of bf16 inputs: one operand
in 16 bits, 2^-16, and the fp32 error; four times that for the decays' gradient.
"""

import math

import pytest
import torch

from mingru_amd import linear_attention, linear_attention_step
from tests.test_linear_attention import inputs, recurrence

pytestmark = pytest.mark.gpu

F32 = 6 * math.sqrt(128) * 2.0**-24
TOL = {torch.float32: F32, torch.bfloat16: 2 * 2.0**-8, torch.float16: F32 + 2.0**-11}
STATE = {torch.float32: F32, torch.bfloat16: F32 + 2.0**-16, torch.float16: F32}


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def off(a, b):
    b = b.detach().double().cpu()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


def check(cuda, B, T, H, Hk, dk, dv, dtype, lengths=None, constant=False, start=True, seed=0,
          layout=lambda t: t, scale=None):
    vals = inputs(B, T, H, Hk, dk, dv, seed, constant=constant)
    vals = [t.to(dtype) for t in vals[:3]] + [t.float() for t in vals[3:]]
    if not start:
        vals.pop()
    ref = [t.double().requires_grad_() for t in vals]
    want = recurrence(*ref[:4], ref[4] if start else None, lengths, scale)
    r = torch.Generator().manual_seed(seed + 1)
    do = torch.randn(B, T, H, dv, generator=r).to(dtype)
    dh = torch.randn(B, H, dk, dv, generator=r)
    wgrads = torch.autograd.grad(want, ref, (do.double(), dh.double()))

    dev = [layout(t.to(cuda)) if i < 3 else t.to(cuda) for i, t in enumerate(vals)]
    dev = [t.requires_grad_() for t in dev]
    L = None if lengths is None else lengths.to(cuda)
    got = linear_attention(*dev[:4], dev[4] if start else None, L, scale)
    grads = torch.autograd.grad(got, dev, (layout(do.to(cuda)), dh.to(cuda)))
    assert got[0].dtype == dtype and got[1].dtype == torch.float32
    errors = {"o": off(got[0], want[0]) / TOL[dtype], "h": off(got[1], want[1]) / STATE[dtype]}
    for n, a, b, w, tol in zip(("q", "k", "v", "g", "h0"), grads, wgrads, vals,
                               (TOL[dtype],) * 3 + (4 * STATE[dtype], STATE[dtype])):
        assert a.shape == w.shape and a.dtype == w.dtype
        errors["d" + n] = off(a, b) / tol
    print({n: round(e, 3) for n, e in errors.items()}, flush=True)
    assert max(errors.values()) <= 1, errors


@pytest.mark.parametrize("dk, dv", [(1, 1), (3, 5), (8, 16), (48, 80), (64, 64), (64, 65), (65, 64),
                                    (64, 128), (128, 64), (128, 128), (100, 120)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_sizes(cuda, dk, dv, dtype):
    check(cuda, 2, 150, 4, 2, dk, dv, dtype, seed=dk)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 128, 129, 517])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(cuda, T, dtype):
    check(cuda, 2, T, 2, 2, 32, 40, dtype, seed=T)


def test_many_sequences(cuda):
    """More workgroups than the chip holds at once: sequences are not cut."""
    check(cuda, 64, 70, 16, 4, 16, 24, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padded_sequences(cuda, dtype):
    T = 300
    lengths = torch.tensor([0, 1, 63, 64, 65, 200, 300], dtype=torch.int32)
    check(cuda, 7, T, 2, 1, 32, 32, dtype, lengths=lengths)
    check(cuda, 7, T, 2, 1, 32, 32, dtype, lengths=lengths.long(), start=False)


def test_padding_is_not_read(cuda):
    q, k, v, g, h = (t.float().to(cuda) for t in inputs(2, 200, 2, 1, 64, 64, documents=False))
    lengths = torch.tensor([200, 70], device=cuda)

    def run():
        ts = [t.clone().requires_grad_() for t in (q, k, v, g, h)]
        o, S = linear_attention(*ts, lengths)
        return o, S, *torch.autograd.grad((o, S), ts, (v, h))

    want = run()
    for t in (q, k, v, g):
        t[1, 70:] = math.nan
    up = v.clone()
    up[1, 70:] = 0
    got = run()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert bool((got[0][1, 70:] == 0).all()) and bool((got[2][1, 70:] == 0).all())


@pytest.mark.parametrize("Hk", [1, 2, 3, 6])
def test_shared_keys(cuda, Hk):
    check(cuda, 1, 100, 6, Hk, 24, 32, torch.bfloat16, seed=Hk)
    check(cuda, 1, 100, 6, Hk, 24, 32, torch.float32, seed=Hk)


def test_one_decay_a_head(cuda):
    check(cuda, 3, 130, 4, 2, 32, 32, torch.float32, constant=True)
    check(cuda, 3, 130, 4, 2, 32, 32, torch.bfloat16, constant=True, start=False)


def test_half_precision(cuda):
    check(cuda, 2, 90, 2, 2, 32, 32, torch.float16)


def _columns(t):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype, device=t.device)
    wide[..., 8:-16] = t
    return wide[..., 8:-16]


def _unaligned(t):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def _heads_first(t):
    return t.transpose(1, 2).contiguous().transpose(1, 2)


def _features_first(t):
    return t.transpose(1, 3).contiguous().transpose(1, 3)


@pytest.mark.parametrize("layout", [_columns, _unaligned, _heads_first, _features_first])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(cuda, layout, dtype):
    check(cuda, 2, 100, 4, 2, 32, 48, dtype, layout=layout, scale=0.25)


def test_only_one_gradient(cuda):
    ts = [t.float() for t in inputs(2, 100, 2, 1, 16, 16)]
    for which in (0, 1):
        ref = [t.double().requires_grad_() for t in ts]
        want = torch.autograd.grad(recurrence(*ref)[which].sin().sum(), ref, allow_unused=True)
        dev = [t.to(cuda).requires_grad_() for t in ts]
        got = torch.autograd.grad(linear_attention(*dev)[which].sin().sum(), dev)
        for a, b in zip(got, want):
            if b is None:
                assert float(a.abs().max()) == 0
            else:
                assert off(a, b) <= 8 * F32


def test_strong_decays(cuda):
    """Factors down to the smallest, whose sums over a chunk reach thousands."""
    q, k, v, g, h = inputs(2, 200, 2, 1, 32, 32, documents=False)
    g = 60 * g
    ref = recurrence(*(t.float().double() for t in (q, k, v, g, h)))
    got = linear_attention(*(t.float().to(cuda) for t in (q, k, v, g, h)))
    for a, b in zip(got, ref):
        assert off(a, b) <= F32


def test_same_on_every_run(cuda):
    vals = inputs(2, 300, 4, 2, 64, 64)
    ts = [t.bfloat16().to(cuda) for t in vals[:3]] + [t.float().to(cuda) for t in vals[3:]]
    ts = [t.requires_grad_() for t in ts]

    def once():
        o, S = linear_attention(*ts)
        return o, S, *torch.autograd.grad((o, S), ts, (torch.ones_like(o), torch.ones_like(S)))

    assert all(torch.equal(a, b) for a, b in zip(once(), once()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk, dv", [(1, 1), (24, 37), (128, 128), (160, 72)])
def test_steps(cuda, dtype, dk, dv):
    q, k, v, g, h = inputs(3, 5, 4, 2, dk, dv)
    q, k, v, g, h = *(t.to(dtype) for t in (q, k, v)), g.float(), h.float()
    want, _ = recurrence(*(t.double() for t in (q, k, v, g, h)))
    S = h.to(cuda)
    for t in range(5):
        before = S.clone()
        ot, S2 = linear_attention_step(*(x[:, t].to(cuda) for x in (q, k, v, g)), S)
        assert torch.equal(S, before)
        S = S2
        assert ot.dtype == dtype and off(ot, want[:, t]) <= TOL[dtype]
    _, S5 = recurrence(*(t.double() for t in (q, k, v, g, h)))
    assert off(S, S5) <= F32


def test_step_layouts(cuda):
    q, k, v, g, h = (t.float().to(cuda) for t in inputs(3, 1, 4, 2, 16, 32))
    want, wS = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], h)
    for f in (lambda t: _columns(t), lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)):
        got, S = linear_attention_step(f(q[:, 0]), f(k[:, 0]), f(v[:, 0]), g[:, 0], f(h))
        assert torch.equal(got, want) and torch.equal(S, wS)
    o, S = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[0, 0])
    wo, wS = recurrence(*(t.double().cpu() for t in (q, k, v)), g[0, 0].double().cpu())
    assert off(o, wo[:, 0]) <= F32 and off(S, wS) <= F32


def test_other_stream_and_graph(cuda):
    ts = [t.float().to(cuda).requires_grad_() for t in inputs(2, 150, 2, 1, 64, 64)]

    up = [ts[i].detach().clone() for i in (2, 4)]

    def step():
        # Nothing that is returned keeps the graph: its leaves' nodes belong to the stream they
        # were made on, and a capture that met nodes of another stream would draw it in.
        o, S = linear_attention(*ts)
        grads = torch.autograd.grad((o, S), ts, up)
        return o.detach(), *grads

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            ts[0].add_(0.25)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


def test_past_32_bits(cuda):
    """More than 2^31 elements of v and o: the second half equals a pass of its own."""
    T, H, d = (1 << 19) + 192, 32, 128
    g = torch.full((H,), -0.01, device=cuda)
    r = torch.Generator(device=cuda).manual_seed(1)
    q = torch.randn(1, T, 1, 16, device=cuda, generator=r, dtype=torch.bfloat16)
    v = torch.randn(1, T, H, d, device=cuda, generator=r, dtype=torch.bfloat16)
    assert v.numel() > 2**31
    o, S = linear_attention(q, q, v, g)
    half = 1 << 18
    o1, S1 = linear_attention(q[:, :half], q[:, :half], v[:, :half], g)
    o2, S2 = linear_attention(q[:, half:], q[:, half:], v[:, half:], g, S1)
    assert off(S, S2) <= 2 * STATE[torch.bfloat16]
    for a, b in ((o[:, : half], o1), (o[:, half:], o2)):
        a, b = a[:, -5000:].float(), b[:, -5000:].float()
        assert off(a, b) <= 2 * TOL[torch.bfloat16]


def test_declines(cuda, monkeypatch):
    ts = [t.float().to(cuda) for t in inputs(1, 5, 1, 1, 130, 4)]
    with pytest.raises(RuntimeError, match="128"):
        linear_attention(*ts)
    with pytest.raises(RuntimeError, match="float64"):
        linear_attention(*(t.to(cuda) for t in inputs(1, 5, 1, 1, 4, 4)))
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    with pytest.warns(UserWarning, match="linear_attention"):
        o, S = linear_attention(*ts)
    wo, wS = recurrence(*(t.double().cpu() for t in ts))
    assert off(o, wo) <= 2 * F32 and off(S, wS) <= 2 * F32
