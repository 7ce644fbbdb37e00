"""What the sequence operators ask of memory, from the C ABI's size entries (no GPU)."""

import os

import pytest

from mingru_amd import _native
from mingru_amd import build as hip_build


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(hip_build.LIB_PATH):
        hip_build.build()
    return _native.load()


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("D", [512, 1024, 4096])
@pytest.mark.parametrize("V", [32768, 128256, 1 << 19])
@pytest.mark.parametrize("N", [4096, 16384, 65536, 131072, 262144])
def test_loss_backward_does_not_grow_with_the_vocabulary(lib, dtype, N, V, D):
    """A piece of d in half a gigabyte (or 512 columns of it), dx and the rows it is summed from a few
    times in fp32, parts of a piece of dW for the workgroups that the chip holds: nothing that grows
    with rows times vocabulary."""
    planes = 2 - dtype
    d = max(1 << 29, 512 * 2 * planes * N)
    ws = lib.mg_vocab_loss_bwd_workspace_bytes(dtype, N, V, D)
    assert ws <= d + 4 * (4 * N * D) + (1 << 29), (ws, d)
    if N * V >= 1 << 32:  # what it is there for: the logits' own bytes are far more
        assert ws <= N * V * 4 / 2 + 4 * (4 * N * D), ws


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("N, V, D", [(64, 50257, 768), (4096, 32768, 1024), (262144, 128256, 4096)])
def test_loss_backward_without_dx_lacks_its_part(lib, dtype, N, V, D):
    whole = lib.mg_vocab_loss_bwd_workspace_bytes(dtype, N, V, D)
    dx = lib.mg_vocab_loss_bwd_dx_bytes(dtype, N, V, D)
    assert 4 * N * D <= dx < whole
    P = 4096  # never followed by the refused calls
    call = lambda to, nbytes: lib.mg_vocab_loss_bwd(  # noqa: E731
        dtype, P, None, P, 1, to, P, None, N, V, D, P, P, nbytes, None)
    assert call(P, whole - 1) == 3
    assert call(None, whole - dx - 1) == 3
