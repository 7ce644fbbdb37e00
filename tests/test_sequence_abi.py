"""The C entries of residual_norm, linear_attention and linear_cross_entropy refuse what they do not
take on the host: null pointers, sizes out of range (status 1), short workspaces (status 3).  No
kernel is launched here; the pointers are never followed."""

import ctypes
import os

import pytest

from mingru_amd import _native
from mingru_amd import build as hip_build

NULL, P = None, 4096  # a pointer that no refused call follows
STRIDES = (ctypes.c_int64 * 15)(*[1] * 15)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(hip_build.LIB_PATH):
        hip_build.build()
    return _native.load()


def replaced(args, **by):
    names = list(args)
    assert set(by) <= set(names)
    return [by.get(n, args[n]) for n in names]


ATTENTION = dict(B=2, T=100, H=4, Hk=2, dk=32, dv=48)
BAD_ATTENTION = [dict(dtype=2), dict(B=0), dict(T=0), dict(H=0), dict(Hk=0), dict(Hk=3),
                 dict(dk=0), dict(dv=0), dict(dk=129), dict(dv=129), dict(H=1 << 17)]


def attention(kind):
    pointers = {"fwd": "q k v g strides lengths h0 o hT state", "bwd": "q k v g do strides lengths "
                "h0 hT state dhT dq dk_ dv_ dg dh0"}[kind].split()
    args = dict(dtype=0, **{p: P for p in pointers})
    args["strides"] = STRIDES
    if kind == "fwd":
        args["bytes"] = 1 << 40
    args |= ATTENTION | dict(scale=1.0)
    if kind == "bwd":
        args |= dict(ws=P, bytes=1 << 40)
    return args | dict(stream=NULL)


@pytest.mark.parametrize("kind", ["fwd", "bwd"])
def test_attention(lib, kind):
    call, args = getattr(lib, f"mg_linear_attention_{kind}"), attention(kind)
    for bad in BAD_ATTENTION:
        assert call(*replaced(args, **bad)) == 1, bad
    optional = {"lengths", "h0", "dhT", "dh0", "stream"}
    for name, value in args.items():
        if (value is P or value is STRIDES) and name not in optional:
            assert call(*replaced(args, **{name: NULL})) == 1, name
    assert call(*replaced(args, bytes=0)) == 3


def test_attention_sizes(lib):
    order = ("dtype", "B", "T", "H", "Hk", "dk", "dv")
    for f in (lib.mg_linear_attention_state_bytes, lib.mg_linear_attention_workspace_bytes):
        good = dict(dtype=0) | ATTENTION
        assert f(*(good[n] for n in order)) > 0
        for bad in BAD_ATTENTION:
            assert f(*((good | bad)[n] for n in order)) == 0, bad


def test_attention_step(lib):
    args = dict(dtype=0, q=P, k=P, v=P, g=P, strides=STRIDES, h=P, o=P, h_out=P, B=2, H=4, Hk=2,
                dk=32, dv=48, scale=1.0, stream=NULL)
    for bad in (dict(dtype=2), dict(B=0), dict(H=0), dict(Hk=3), dict(dk=0), dict(dv=0),
                *(dict([(n, NULL)]) for n in "q k v g strides h o h_out".split())):
        assert lib.mg_linear_attention_step(*replaced(args, **bad)) == 1, bad


LOSS = dict(N=10, V=100, D=16)
BAD_LOSS = [dict(dtype=2), dict(N=0), dict(V=0), dict(D=0), dict(N=(1 << 30) + 1),
            dict(V=(1 << 30) + 1), dict(D=(1 << 20) + 1)]


@pytest.mark.parametrize("N", [10, 1000])  # both families of kernels
@pytest.mark.parametrize("dtype", [0, 1])
def test_loss(lib, dtype, N):
    fwd = dict(dtype=dtype, x=P, ldx=16, w=P, bias=NULL, target=P, ignore=-100, reduction=1,
               loss=P) | LOSS | dict(state=P, state_bytes=1 << 40, ws=P, bytes=1 << 40, stream=NULL)
    bwd = dict(dtype=dtype, w=P, bias=NULL, dloss=P, reduction=1, dx=P, dw=P, db=NULL) | LOSS | dict(
        state=P, ws=P, bytes=1 << 40, stream=NULL)
    for args, call, needed in ((fwd, lib.mg_vocab_loss_fwd, "x w target loss state ws"),
                               (bwd, lib.mg_vocab_loss_bwd, "w dloss state ws")):
        args["N"] = N
        for bad in (*BAD_LOSS, dict(reduction=-1), dict(reduction=3),
                    *(dict([(n, NULL)]) for n in needed.split())):
            assert call(*replaced(args, **bad)) == 1, bad
        assert call(*replaced(args, bytes=0)) == 3
    assert lib.mg_vocab_loss_fwd(*replaced(fwd, ldx=15)) == 1
    assert lib.mg_vocab_loss_fwd(*replaced(fwd, state_bytes=0)) == 3
    assert lib.mg_vocab_loss_bwd(*replaced(bwd, dw=NULL, db=P)) == 1
    for f in (lib.mg_vocab_loss_state_bytes, lib.mg_vocab_loss_fwd_workspace_bytes,
              lib.mg_vocab_loss_bwd_workspace_bytes):
        good = dict(dtype=dtype) | LOSS | dict(N=N)
        assert f(*good.values()) > 0
        for bad in BAD_LOSS:
            assert f(*(good | bad).values()) == 0, bad


def test_norm(lib):
    fwd = dict(dtype=0, pdtype=0, post=2, act=1, pre=1, h=P, ldh=64, x=P, ldx=64, gate=P, ldg=64,
               scale=P, scale_const=1.0, post_w=P, post_b=NULL, pre_w=P, pre_b=P, r=P, y=P, stats=P,
               rows=10, D=64, eps=1e-5, stream=NULL)
    for bad in (dict(post=3), dict(act=3), dict(pre=3), dict(dtype=2), dict(h=NULL), dict(gate=NULL),
                dict(y=NULL), dict(ldh=63), dict(ldx=63), dict(ldg=63), dict(D=0), dict(D=8193),
                dict(rows=0)):
        assert lib.mg_residual_norm_fwd(*replaced(fwd, **bad)) == 1, bad
    assert lib.mg_residual_norm_workspace_bytes(10, 64) > 0
    assert lib.mg_residual_norm_workspace_bytes(0, 64) == 0
    assert lib.mg_residual_norm_workspace_bytes(10, 8193) == 0
