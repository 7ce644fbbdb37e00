"""The C entries of the paged cache and of beam search refuse what they do not take on the host:
null pointers, sizes out of range (status 1), short workspaces (status 3), launches past the grid
(status 4).  No kernel is launched here; the pointers are never followed."""

import ctypes
import os

import pytest

from mingru_amd import _native
from mingru_amd import build as hip_build

NULL, P = None, 4096  # a pointer that no refused call follows
STRIDES = (ctypes.c_int64 * 16)(*[1] * 16)


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(hip_build.LIB_PATH):
        hip_build.build()
    return _native.load()


def replaced(args, **by):
    assert set(by) <= set(args)
    return [by.get(n, args[n]) for n in args]


def check(call, args, bad, optional):
    for change in bad:
        assert call(*replaced(args, **change)) == 1, change
    for name, value in args.items():
        if (value is P or value is STRIDES) and name not in optional:
            assert call(*replaced(args, **{name: NULL})) == 1, name


def test_append(lib):
    args = dict(dtype=0, q=P, k=P, v=P, k_cache=P, v_cache=P, q_out=P, strides=STRIDES, ints=0,
                pages=P, start=P, lengths=P, freq_dtype=0, freq=P, n=4, interleaved=0, B=2, T=3,
                H=4, Hk=2, dk=8, dv=8, N=5, M=2, P=4, stream=NULL)
    bad = [dict(dtype=3), dict(dtype=-1), dict(ints=8), dict(ints=-1), dict(B=0), dict(T=0),
           dict(H=0), dict(Hk=0), dict(dk=0), dict(dv=0), dict(N=0), dict(M=0), dict(P=0),
           dict(P=1 << 31), dict(n=-1), dict(n=5), dict(freq_dtype=2), dict(T=1 << 40),
           dict(B=1 << 40), dict(dk=1 << 24, H=8), dict(n=1025, dk=4096)]
    check(lib.mg_paged_append, args, bad, {"q", "lengths", "stream"})
    assert lib.mg_paged_append(*replaced(args, B=1 << 30, T=100)) == 4


ATTEND = dict(B=2, H=4, Hk=2, dk=8, dv=8, M=3, P=4)
BAD = [dict(B=0), dict(H=0), dict(Hk=0), dict(Hk=3), dict(dk=0), dict(dv=0), dict(dk=257),
       dict(dv=257), dict(M=0), dict(P=0), dict(M=1 << 31), dict(P=1 << 31), dict(B=1 << 24),
       dict(M=1 << 16, P=1 << 15), dict(B=1 << 20, H=16, Hk=16)]


def test_attention(lib):
    args = dict(dtype=1, q=P, k_cache=P, v_cache=P, strides=STRIDES, ints=0, pages=P, lengths=P, o=P,
                B=2, H=4, Hk=2, dk=8, dv=8, N=5, M=3, P=4, window=0, scale=1.0, ws=P,
                bytes=1 << 40, stream=NULL)
    bad = [*BAD, dict(dtype=3), dict(dtype=-1), dict(ints=4), dict(ints=-1), dict(N=0),
           dict(N=1 << 31), dict(window=-1)]
    check(lib.mg_paged_attention_step, args, bad, {"stream"})
    assert lib.mg_paged_attention_step(*replaced(args, bytes=0)) == 3
    size = lib.mg_paged_attention_workspace_bytes
    for dtype in (0, 1, 2):
        assert size(dtype, *ATTEND.values()) > 0
        for change in BAD:
            assert size(dtype, *replaced(ATTEND, **change)) == 0, change
    assert size(3, *ATTEND.values()) == size(-1, *ATTEND.values()) == 0


SELECT = dict(B=2, K=3, V=50, W=4)
BAD_SELECT = [dict(B=0), dict(K=0), dict(V=0), dict(W=0), dict(W=65), dict(K=257), dict(V=1 << 30),
              dict(K=1, V=3), dict(B=1 << 22), dict(K=200, V=1 << 24)]


def test_select(lib):
    args = dict(dtype=0, logits=P, scores=P, finished=P, strides=STRIDES, end=1, out=P, parents=P,
                tokens=P, done=P, **SELECT, ws=P, bytes=1 << 40, stream=NULL)
    bad = [*BAD_SELECT, dict(dtype=3), dict(dtype=-1), dict(end=50), dict(end=-1)]
    check(lib.mg_beam_select, args, bad, {"finished", "done", "stream"})
    assert lib.mg_beam_select(*replaced(args, end=-1, done=NULL)) == 1  # finished without an end
    assert lib.mg_beam_select(*replaced(args, bytes=0)) == 3
    size = lib.mg_beam_select_workspace_bytes
    assert size(0, *SELECT.values()) > 0 and size(3, *SELECT.values()) == 0
    for change in BAD_SELECT:
        assert size(0, *replaced(SELECT, **change)) == 0, change


def test_reorder(lib):
    pointers = (ctypes.c_void_p * 2)(P, P)
    sizes = (ctypes.c_int64 * 2)(8, 8)
    args = dict(count=2, src=pointers, dst=pointers, strides=sizes, bytes=sizes, wide=0, parents=P,
                pb=1, pw=1, B=2, K=3, W=4, stream=NULL)
    call = lib.mg_reorder_rows
    bad = [dict(count=0), dict(src=NULL), dict(dst=NULL), dict(strides=NULL), dict(bytes=NULL),
           dict(wide=2), dict(B=0), dict(K=0), dict(W=0), dict(B=1 << 31), dict(W=1 << 31),
           dict(B=1 << 16, W=1 << 15), dict(K=1 << 31),
           dict(src=(ctypes.c_void_p * 2)(P, None)), dict(dst=(ctypes.c_void_p * 2)(None, P)),
           dict(bytes=(ctypes.c_int64 * 2)(8, 0)), dict(bytes=(ctypes.c_int64 * 2)(1 << 40, 8))]
    check(call, args, bad, {"stream"})
    assert call(*replaced(args, bytes=(ctypes.c_int64 * 2)(1 << 38, 8), B=1 << 10, W=1 << 10)) == 4
