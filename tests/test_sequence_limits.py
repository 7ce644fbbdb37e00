"""Sizes whose launches would pass 2^32 threads are refused by the C entries before any launch, and
declined before the call (CPU)."""

import ctypes

import pytest
import torch

from mingru_amd import hip_scans, hip_sequence
from tests.test_sequence_workspace import lib  # noqa: F401


def test_attention_pairs(lib):  # noqa: F811
    for f in (lib.mg_linear_attention_state_bytes, lib.mg_linear_attention_workspace_bytes):
        for B, H in ((1 << 21, 4), (1 << 23, 1), (1 << 62, 4)):
            assert f(0, B, 1, H, 1, 4, 4) == 0
        assert f(0, (1 << 21) - 1, 1, 4, 1, 4, 4) > 0
    strides = (ctypes.c_int64 * 15)(*[1] * 15)
    P = 4096  # never followed
    step = lambda B, H: lib.mg_linear_attention_step(  # noqa: E731
        0, P, P, P, P, strides, P, P, P, B, H, 1, 4, 4, 1.0, None)
    assert step(1 << 22, 4) == 1 and step(1 << 24, 1) == 1 and step(1 << 62, 4) == 1


def test_attention_declines_them():
    B = 1 << 21
    q, g = torch.zeros(1, 1, 1, 4).expand(B, 1, 1, 4), torch.zeros(4)
    v = torch.zeros(1, 1, 4, 4).expand(B, 1, 4, 4)
    with pytest.raises(hip_scans.ScanFallback, match="2\\^23"):
        hip_sequence.linear_attention_impl(q, q, v, g, None, None, 1.0)
    q, v = (t[:1, 0].expand(1 << 22, *t.shape[2:]) for t in (q, v))
    h = torch.zeros(1, 4, 4, 4).expand(1 << 22, 4, 4, 4)
    with pytest.raises(hip_scans.ScanFallback, match="2\\^24"):
        hip_sequence.linear_attention_step_impl(q, q, v, g, h, 1.0)
