"""``DecayLM.generate`` refuses lengths that leave no last token, or name one past the prompt, on the
host: the first took the last padding token for the prompt's, the second indexed out of range."""

import pytest
import torch

from mingru_amd.decay_lm import DecayLM


@pytest.mark.parametrize("lengths", [[0, 3], [-1, 3], [6, 3]])
def test_lengths_out_of_range(lengths):
    torch.manual_seed(0)
    model, prompt = DecayLM(11, 16, 1, 2), torch.randint(0, 11, (2, 5))
    with pytest.raises(ValueError, match="lengths"):
        model.generate(prompt, 2, torch.tensor(lengths))
    with pytest.raises(ValueError, match="prompt"):
        model.generate(prompt[:, :0], 2)
    assert model.generate(prompt, 2, torch.tensor([1, 5])).shape == (2, 2)
