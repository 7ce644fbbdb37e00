"""``residual_norm`` kernels against the definition in float64: every kind of norm and gate,
row widths around each lane group's, strides, missing gradients, streams and graphs.

Tolerances, as the 2-norm of the difference over the 2-norm of the result.  fp32: an element
passes about 40 roundings of 2^-24 on its way (two norms' sums over at most 16 elements a lane
and a tree of lanes, exp, division, products), independent ones: 40 * 2^-24 = 2.4e-6.  bf16:
the same and one rounding of the result to 8 significant bits, 2^-8 at most.
"""

import pytest
import torch

from mingru_amd import residual_norm
from tests.test_residual_norm import inputs, plain

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 40 * 2.0**-24, torch.bfloat16: 2.0**-8 + 40 * 2.0**-24,
       torch.float16: 2.0**-11 + 40 * 2.0**-24}
NAMES = ("h", "x", "gate", "scale", "post_weight", "post_bias", "pre_weight", "pre_bias")


@pytest.fixture(autouse=True)
def _hip(monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")


def off(a, b):
    b = b.double()
    b = b.detach()
    return float((a.detach().double().cpu() - b).norm() / b.norm().clamp(min=1e-300))


def check(cuda, shape, dtype, post, act, pre, stream=True, seed=0, vdtype=None, layout=None,
          tol=None):
    vals = dict(zip(NAMES, inputs(shape, seed)))
    for n in NAMES:
        vals[n] = vals[n].to(dtype if n in NAMES[:3] else vdtype or dtype)
    if act is None:
        vals["gate"] = None
    if not stream:
        vals["x"] = vals["scale"] = None
    if post == "none":
        vals["post_weight"] = vals["post_bias"] = None
    if pre == "none":
        vals["pre_weight"] = vals["pre_bias"] = None
    used = [n for n in NAMES if vals[n] is not None]
    ref = {n: vals[n].double().requires_grad_() for n in used}
    at = {n: ref.get(n) for n in NAMES}
    want = plain(at["h"], at["x"], post, at["post_weight"], at["post_bias"], at["gate"], act,
                 at["scale"], pre, at["pre_weight"], at["pre_bias"])
    g = torch.Generator().manual_seed(seed + 100)
    ups = [torch.randn(*shape, generator=g).to(dtype) for _ in want]
    wgrads = torch.autograd.grad(want, [ref[n] for n in used], [u.double() for u in ups])

    dev = {n: vals[n].to(cuda) for n in used}
    if layout is not None:
        dev = {n: layout(t) if n in NAMES[:3] else t for n, t in dev.items()}
        ups = [layout(u.to(cuda)) for u in ups]
    dev = {n: t.requires_grad_() for n, t in dev.items()}
    kw = {n: dev.get(n) for n in NAMES[2:]}
    got = residual_norm(dev["h"], dev.get("x"), post=post, pre=pre, gate_act=act or "silu", **kw)
    got = got if isinstance(got, tuple) else (got,)
    grads = torch.autograd.grad(got, [dev[n] for n in used], [u.to(cuda) for u in ups])
    for name, a, b in zip(("r", "y"), got, want):
        assert a.dtype == dtype and off(a, b) <= (tol or TOL[dtype]), (name, off(a, b))
    for n, a, b in zip(used, grads, wgrads):
        assert a.dtype == vals[n].dtype and a.shape == vals[n].shape
        # A sum over the rows of a row vector's gradient adds its own rounding error, but no
        # more than as many roundings of its partial sums.
        assert off(a, b) <= 2 * (tol or TOL[vals[n].dtype]), (n, off(a, b))


@pytest.mark.parametrize("post", ["none", "layer", "rms"])
@pytest.mark.parametrize("act", [None, "sigmoid", "silu"])
@pytest.mark.parametrize("pre", ["none", "layer", "rms"])
@pytest.mark.parametrize("stream", [True, False])
def test_kinds(cuda, post, act, pre, stream):
    check(cuda, (3, 5, 40), torch.float32, post, act, pre, stream)


@pytest.mark.parametrize("D", [1, 2, 7, 16, 127, 128, 129, 248, 256, 257, 512, 513, 1000, 1024,
                               1025, 2048, 2056, 4096, 4104, 8191, 8192])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths(cuda, D, dtype):
    # A row of one or two elements has a near-singular LayerNorm: its own RMS norm instead.
    check(cuda, (19, D), dtype, "rms", "sigmoid", "layer" if D > 2 else "rms", seed=D,
          vdtype=torch.float32)


@pytest.mark.parametrize("rows", [1, 2, 15, 17, 4099])
def test_rows(cuda, rows):
    check(cuda, (rows, 96), torch.float32, "layer", "silu", "rms", seed=rows)


def test_types(cuda):
    check(cuda, (33, 72), torch.bfloat16, "layer", "silu", "rms")
    check(cuda, (33, 72), torch.float16, "layer", "silu", "rms")


def _columns(t):
    """Rows inside wider ones, as columns of a joined projection are."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 24, dtype=t.dtype, device=t.device)
    wide[..., 8:-16] = t
    return wide[..., 8:-16]


def _unaligned(t):
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def _turned(t):
    return t.transpose(0, -1).contiguous().transpose(0, -1)


@pytest.mark.parametrize("layout", [_columns, _unaligned, _turned])
def test_strides(cuda, layout):
    check(cuda, (6, 4, 64), torch.bfloat16, "rms", "silu", "layer", layout=layout)


def test_gate_of_each_sequence(cuda):
    """A gate broadcast over the time axis gets its own gradient, summed over it."""
    h, x, gate = (t.float() for t in inputs((2, 9, 48))[:3])
    gate = gate[:, :1].contiguous()
    out = []
    for dev, up in (("cpu", torch.float64), (cuda, torch.float32)):
        ts = [t.to(dev, up).requires_grad_() for t in (h, x, gate)]
        r = residual_norm(ts[0], ts[1], gate=ts[2], gate_act="sigmoid", pre="none") \
            if dev != "cpu" else ts[1] + ts[0] * torch.sigmoid(ts[2])
        out.append(torch.autograd.grad(r.square().sum(), ts))
    for a, b in zip(out[1], out[0]):
        assert a.shape == b.shape and off(a, b) <= 2 * TOL[torch.float32]


def test_missing_gradients(cuda):
    """Only one output used, and only some inputs asked for."""
    h, x, gate, scale, pw, pb, qw, qb = (t.float() for t in inputs((7, 40)))
    for use in (0, 1):
        for asked in (["h"], ["x"], ["pre_weight"], ["h", "x"]):
            got = []
            for dev, up in (("cpu", torch.float64), (cuda, torch.float32)):
                ts = {"h": h, "x": x, "pre_weight": qw}
                ts = {n: t.to(dev, up).requires_grad_(n in asked) for n, t in ts.items()}
                out = (plain(ts["h"], ts["x"], "none", None, None, None, None, None, "layer",
                             ts["pre_weight"], None) if dev == "cpu" else
                       residual_norm(ts["h"], ts["x"], pre_weight=ts["pre_weight"]))
                if not out[use].requires_grad:
                    got.append([])
                    continue
                got.append(torch.autograd.grad(out[use].sin().sum(), [ts[n] for n in asked],
                                               allow_unused=True))
            for a, b in zip(*got[::-1]):
                assert (a is None or float(a.abs().max()) == 0) if b is None \
                    else off(a, b) <= 4 * TOL[torch.float32]


def test_same_on_every_run(cuda):
    """Row vectors' gradients are added in one order."""
    ts = [t.float().to(cuda).requires_grad_() for t in inputs((5000, 136))]

    def once():
        r, y = residual_norm(ts[0], ts[1], post="rms", gate=ts[2], scale=ts[3],
                             post_weight=ts[4], pre_weight=ts[6], pre_bias=ts[7])
        return torch.autograd.grad((r.square() + y).sum(), [ts[i] for i in (0, 1, 2, 3, 4, 6, 7)])

    a, b = once(), once()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_other_stream_and_graph(cuda):
    h, x, gate = (t.float().to(cuda) for t in inputs((64, 512))[:3])
    want = residual_norm(h, x, post="rms", gate=gate)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = residual_norm(h, x, post="rms", gate=gate)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    ts = [t.clone().requires_grad_() for t in (h, x, gate)]
    w = torch.ones(512, device=cuda, requires_grad=True)

    def step():
        r, y = residual_norm(ts[0], ts[1], post="rms", post_weight=w, gate=ts[2])
        return torch.autograd.grad((r, y), (*ts, w), (h, x))

    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            ts[0].add_(0.5)
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i


def test_special_values(cuda):
    """Constant rows, rows of zeros, and a NaN or infinity that stays in its own row."""
    h = torch.randn(6, 64, device=cuda)
    h[0], h[1] = 0.0, 3.0
    h[2, 5], h[3, 5] = float("nan"), float("inf")
    r, y = residual_norm(h, torch.zeros_like(h), post="layer", pre="rms")
    assert bool((r[:2] == 0).all()) and bool((y[:2] == 0).all())
    assert bool(r[2:4].isnan().all()) and bool(torch.isfinite(r[4:]).all())
    assert bool(torch.isfinite(y[4:]).all())


def test_declines(cuda, monkeypatch):
    wide = torch.randn(2, 8200, device=cuda)
    with pytest.raises(RuntimeError, match="8192"):
        residual_norm(wide)
    with pytest.raises(RuntimeError, match="float64"):
        residual_norm(wide[:, :64].double())
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    with pytest.warns(UserWarning, match="residual_norm"):
        r, y = residual_norm(wide)
    assert off(y, torch.nn.functional.layer_norm(wide.double().cpu(), (8200,))) <= TOL[torch.float32]
