"""``reorder_states`` on the GPU out of states without rows: no parent is one of them, so rows are 0, and the
host looks at no value of the device."""

import pytest
import torch

from mingru_amd import reorder_states

pytestmark = pytest.mark.gpu


def test_rows_are_0(cuda, monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    states = {"a": torch.empty(0, 3, device=cuda), "b": [torch.empty(0, dtype=torch.int32, device=cuda), None]}
    parents = torch.tensor([[0, -1, 2], [1, 0, 0]], device=cuda)
    got = reorder_states(states, parents)
    assert got["a"].shape == (6, 3) and not bool(got["a"].any()) and got["b"][1] is None
    assert got["b"][0].shape == (6,) and got["b"][0].dtype == torch.int32 and not bool(got["b"][0].any())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = reorder_states(states, parents)
    graph.replay()
    assert not bool(out["a"].any())


def test_no_rows_asked_for(cuda, monkeypatch):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    none = torch.empty(0, 2, dtype=torch.int64, device=cuda)
    assert reorder_states(torch.empty(0, 3, device=cuda), none).shape == (0, 3)
    assert reorder_states(torch.ones(4, 3, device=cuda), none.view(2, 0)).shape == (0, 3)
