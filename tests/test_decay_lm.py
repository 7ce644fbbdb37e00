"""The example model: its one-token form continues its pass, padding does not matter, and it
trains; on the GPU the kernels run it to the CPU's results."""

import pytest
import torch

from mingru_amd.decay_lm import DecayLM, repeated_patterns


def model(seed=0, **kw):
    torch.manual_seed(seed)
    return DecayLM(32, d_model=64, n_layers=2, n_heads=4, n_key_heads=2, **kw)


def check_steps(m, tokens, tol):
    want, states = m(tokens)
    x, y = None, None
    state = [None] * len(m.blocks)
    with torch.no_grad():
        for t in range(tokens.shape[1]):
            x, y = m._enter(tokens[:, t])
            for i, block in enumerate(m.blocks):
                x, y, state[i] = block.step(x, y, state[i])
            assert torch.allclose(y, want[:, t], rtol=tol, atol=tol), t
    for a, b in zip(state, states):
        assert torch.allclose(a, b, rtol=tol, atol=tol)


def test_steps_continue_the_pass():
    g = torch.Generator().manual_seed(1)
    check_steps(model().double(), torch.randint(0, 32, (2, 12), generator=g), 1e-9)


def test_padded_prompts_generate_as_their_own():
    m = model().double()
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 32, (3, 10), generator=g)
    lengths = torch.tensor([10, 4, 1])
    got = m.generate(tokens, 5, lengths)
    for row, n in enumerate(lengths.tolist()):
        assert torch.equal(got[row : row + 1], m.generate(tokens[row : row + 1, :n], 5))


def test_refusals():
    with pytest.raises(ValueError, match="n_heads"):
        DecayLM(32, d_model=66, n_heads=4)
    with pytest.raises(ValueError, match="n_key_heads"):
        DecayLM(32, d_model=64, n_heads=4, n_key_heads=3)


def train(m, steps, device):
    """Losses of steps on one batch, which a model that learns at all comes to know."""
    g = torch.Generator(device=device).manual_seed(3)
    tokens = repeated_patterns(4, 32, 6, 32, g, device)
    optimizer = torch.optim.AdamW(m.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        loss = m.loss(tokens)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def test_trains():
    losses = train(model(), 60, "cpu")
    assert losses[-1] < 0.5 * losses[0]


@pytest.mark.gpu
def test_gpu_gradients_match_the_cpu(cuda, monkeypatch):
    """Loss and every parameter's gradient against the eager bodies in float64."""
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    m = model()
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, 32, (3, 150), generator=g)
    tokens[1, 90:] = -100
    monkeypatch.setenv("MINGRU_SCAN", "auto")
    ref = model().double()
    want = ref.loss(tokens)
    want.backward()
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    m = m.to(cuda)
    loss = m.loss(tokens.to(cuda))
    loss.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    for (name, a), b in zip(m.named_parameters(), ref.parameters()):
        off = (a.grad.double().cpu() - b.grad).norm() / b.grad.norm()
        # About ten operators in a row, each 4e-6 at most off.
        assert float(off) <= 4e-5, (name, float(off))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gpu_trains_and_generates(cuda, monkeypatch, dtype):
    monkeypatch.setenv("MINGRU_SCAN", "hip")
    m = model().to(cuda, dtype)
    losses = train(m, 60, "cuda")
    assert losses[-1] < 0.5 * losses[0]
    tokens = repeated_patterns(8, 30, 6, 32, torch.Generator(device="cuda").manual_seed(5), "cuda")
    assert m.generate(tokens[:, :24], 6).shape == (8, 6)
    if dtype == torch.float32:
        with torch.no_grad():
            check_steps(m, tokens[:, :12], 1e-4)
