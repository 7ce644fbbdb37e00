"""A small language model of the operators in :mod:`mingru_amd.sequence_ops`, as an example of
using them together: blocks of decaying linear attention and an MLP between fused norms, trained
with the vocabulary loss and generating through the one-token forms.

``python -m mingru_amd.decay_lm`` trains it on a synthetic task (a random pattern repeated, which
a model can only continue by recalling it) and prints the losses and a generated continuation.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn as nn
import torch.nn.functional as F

from .sequence_ops import (
    linear_attention,
    linear_attention_step,
    linear_cross_entropy,
    residual_norm,
)

__all__ = ["DecayBlock", "DecayLM"]


class DecayBlock(nn.Module):
    """Attention with a decay for each token and head, then an MLP.

    ``forward`` and ``step`` take the residual stream and its norm for this block, and return
    both for the next one: each addition to the stream and the norm that follows it are one
    ``residual_norm``.
    """

    def __init__(self, d_model: int, n_heads: int, n_key_heads: int | None = None,
                 mlp_expansion: int = 4):
        super().__init__()
        n_key_heads = n_heads if n_key_heads is None else n_key_heads
        if d_model % n_heads or n_heads % n_key_heads:
            raise ValueError(f"d_model ({d_model}) must be a multiple of n_heads ({n_heads}), and "
                             f"n_heads of n_key_heads ({n_key_heads})")
        self.H, self.Hk, self.d = n_heads, n_key_heads, d_model // n_heads
        self.widths = (self.Hk * self.d, self.Hk * self.d, d_model, d_model, n_heads)
        self.proj = nn.Linear(d_model, sum(self.widths), bias=False)
        self.decay_bias = nn.Parameter(torch.linspace(-4.0, 0.0, n_heads))
        self.head_norm = nn.Parameter(torch.ones(self.d))
        self.out = nn.Linear(d_model, d_model, bias=False)
        self.scale = nn.Parameter(torch.ones(d_model))
        self.mlp_norm = nn.Parameter(torch.ones(d_model))
        self.up = nn.Linear(d_model, mlp_expansion * d_model)
        self.down = nn.Linear(mlp_expansion * d_model, d_model)
        self.next_norm = nn.Parameter(torch.ones(d_model))

    def _heads(self, y):
        """Queries, keys, values, gates (..., heads, d) and log decays (..., heads)."""
        q, k, v, gate, decay = self.proj(y).split(self.widths, -1)
        q, k, v, gate = (t.unflatten(-1, (-1, self.d)) for t in (q, k, v, gate))
        # A decay near 1 is a log decay near 0 only in 32 bits or more.
        wide = torch.promote_types(decay.dtype, torch.float32)
        return q, k, v, gate, -F.softplus(decay.to(wide) + self.decay_bias.to(wide))

    def _join(self, x, o, gate):
        h = residual_norm(o, post="rms", post_weight=self.head_norm, gate=gate, pre="none")
        x, y = residual_norm(self.out(h.flatten(-2)), x, scale=self.scale, pre="rms",
                             pre_weight=self.mlp_norm)
        h = self.down(F.gelu(self.up(y)))
        return residual_norm(h, x, pre="rms", pre_weight=self.next_norm)

    def forward(self, x, y, state=None, lengths=None):
        q, k, v, gate, decay = self._heads(y)
        o, state = linear_attention(q, k, v, decay, state, lengths)
        return (*self._join(x, o, gate), state)

    def step(self, x_t, y_t, state=None):
        q, k, v, gate, decay = self._heads(y_t)
        o, state = linear_attention_step(q, k, v, decay, state)
        return (*self._join(x_t, o, gate), state)


class DecayLM(nn.Module):
    """Embedding, ``DecayBlock`` s and a head over the vocabulary."""

    def __init__(self, vocabulary: int, d_model: int = 128, n_layers: int = 2, n_heads: int = 4,
                 n_key_heads: int | None = None):
        super().__init__()
        self.embed = nn.Embedding(vocabulary, d_model)
        self.norm = nn.Parameter(torch.ones(d_model))
        self.blocks = nn.ModuleList(
            DecayBlock(d_model, n_heads, n_key_heads) for _ in range(n_layers))
        self.head = nn.Linear(d_model, vocabulary, bias=False)

    def _enter(self, tokens):
        x = self.embed(tokens)
        return residual_norm(x, pre="rms", pre_weight=self.norm)

    def forward(self, tokens, state=None, lengths=None):
        """Last hidden rows (B, T, d_model), normed, and each block's state."""
        x, y = self._enter(tokens)
        new = []
        for block, h in zip(self.blocks, state or [None] * len(self.blocks)):
            x, y, h = block(x, y, h, lengths)
            new.append(h)
        return y, new

    def loss(self, tokens, ignore_index: int = -100):
        """Mean loss of each token but the first; ``ignore_index`` marks padding at the end."""
        inputs = tokens[:, :-1].clamp(min=0)
        y, _ = self(inputs)
        return linear_cross_entropy(y, self.head.weight, tokens[:, 1:], ignore_index=ignore_index)

    @torch.no_grad()
    def generate(self, prompt, n: int, lengths=None):
        """The ``n`` likeliest next tokens, one after another, after each prompt (B, T), whose
        ``lengths`` (B), of 1 to T tokens, leave off padding at the end."""
        T = prompt.shape[1]
        if T == 0:
            raise ValueError("the prompt has no token to go on from")
        if lengths is not None and bool(((lengths < 1) | (lengths > T)).any()):
            raise ValueError(f"lengths are from 1 to the prompt's {T} tokens (got {lengths.tolist()})")
        y, state = self(prompt, lengths=lengths)
        rows = torch.arange(len(prompt), device=prompt.device)
        y = y[:, -1] if lengths is None else y[rows, lengths.long() - 1]
        out = []
        for _ in range(n):
            token = self.head(y).argmax(-1)
            out.append(token)
            x, y = self._enter(token)
            new = []
            for block, h in zip(self.blocks, state):
                x, y, h = block.step(x, y, h)
                new.append(h)
            state = new
        return torch.stack(out, 1)


def repeated_patterns(batch: int, length: int, period: int, vocabulary: int, generator=None,
                      device="cpu"):
    """Random patterns of ``period`` tokens, each repeated to ``length``."""
    one = torch.randint(0, vocabulary, (batch, period), generator=generator, device=device)
    return one.repeat(1, -(-length // period))[:, :length]


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--steps", type=int, default=2000)
    p.add_argument("--batch", type=int, default=32)
    p.add_argument("--length", type=int, default=64)
    p.add_argument("--vocabulary", type=int, default=64)
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--bf16", action="store_true")
    a = p.parse_args()
    torch.manual_seed(0)
    model = DecayLM(a.vocabulary).to(a.device, torch.bfloat16 if a.bf16 else torch.float32)
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for step in range(a.steps):
        loss = model.loss(repeated_patterns(a.batch, a.length, 8, a.vocabulary, device=a.device))
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        if step % 200 == 0 or step == a.steps - 1:
            print(f"step {step}: loss {loss.item():.3f}", flush=True)
    tokens = repeated_patterns(1, 40, 8, a.vocabulary, device=a.device)
    print("pattern  ", tokens[0, 24:40].tolist())
    print("generated", model.generate(tokens[:, :24], 16)[0].tolist())


if __name__ == "__main__":
    main()
