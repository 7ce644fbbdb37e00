"""``reorder_states`` gives back the classes that it was given."""

import collections
from typing import NamedTuple

import torch

from mingru_amd import reorder_states


class Pair(NamedTuple):
    a: torch.Tensor
    b: object


class Named(dict):
    def __init__(self, name, **kw):
        super().__init__(**kw)
        self.name = name


class Layers(list):
    def __init__(self, name, each):
        super().__init__(each)
        self.name = name


class Row(tuple):
    pass


def test_classes_are_kept():
    x = torch.arange(12.0).view(6, 2)
    parents = torch.tensor([[2, 0, 0], [1, 1, 2]])
    at = torch.tensor([2, 0, 0, 4, 4, 5])
    ordered = collections.OrderedDict([("z", x), ("a", None), ("m", [x + 1])])
    default = collections.defaultdict(list, k=x)
    states = [ordered, default, Named("n", k=x), Layers("l", [x, (x,)]), Row((x, x)), Pair(x, {"y": x}),
              (x, [x]), {"k": x}]
    before = [type(s) for s in states]
    got = reorder_states(states, parents)
    assert type(got) is list and [type(s) for s in got] == before
    assert list(got[0]) == ["z", "a", "m"] and got[0]["a"] is None
    assert torch.equal(got[0]["z"], x[at]) and torch.equal(got[0]["m"][0], x[at] + 1)
    assert torch.equal(got[1]["k"], x[at]) and got[1]["new"] == []
    assert got[2].name == "n" and torch.equal(got[2]["k"], x[at])
    assert got[3].name == "l" and torch.equal(got[3][0], x[at]) and torch.equal(got[3][1][0], x[at])
    assert torch.equal(got[4][1], x[at])
    assert torch.equal(got[5].a, x[at]) and torch.equal(got[5].b["y"], x[at])
    # What was given stays.
    assert ordered["z"] is x and states[2]["k"] is x and states[3][0] is x and "new" not in default
