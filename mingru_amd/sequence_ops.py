"""Operators around the mixers that a language model needs: the norms of a residual block
with its gate and scale, attention with a state that decays, and the loss over a vocabulary.

The reference has none of them; its blocks run torch's LayerNorm and an addition
(``src/mingru/min_gru.py:3819-3872``).  They follow the scans' contract: ``MINGRU_SCAN``
picks the path on every call, GPU tensors run the HIP kernels of
:mod:`mingru_amd.hip_sequence`, a decline falls back to the eager body with a
once-per-process warning (``auto``) or raises ``RuntimeError`` (``hip``), and CPU tensors
run the eager body, which defines the results.
"""

from __future__ import annotations

import warnings

import torch

from .min_gru import _resolve_native_dispatch, _resolve_scan_mode

__all__ = ["residual_norm"]

_warned: set = set()


def _dispatch(what: str, is_cuda: bool, call):
    """``call(hip_sequence)``, or ``None`` for the eager body; the modes' rules as for the scans."""
    mode = _resolve_scan_mode(is_cuda)
    if mode is None:
        return None

    def _call(scans):
        status = scans.available()
        if status is not True:
            raise scans.ScanFallback(str(status))
        from mingru_amd import hip_sequence

        return call(hip_sequence)

    result, reason = _resolve_native_dispatch(mode, what, _call)
    if reason is None:
        return result
    if what not in _warned:
        warnings.warn(f"MINGRU_SCAN=auto ran the eager {what} despite CUDA inputs: {reason}",
                      stacklevel=3)
        _warned.add(what)
    return None


def _wide(t: torch.Tensor) -> torch.Tensor:
    """``t`` in the eager bodies' type: 32 bits at least."""
    return t if t.dtype == torch.float64 else t.float()


def _check_floats(what: str, **tensors) -> None:
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not torch.is_tensor(t) or not t.dtype.is_floating_point:
            raise TypeError(f"{what}: {name} must be a floating-point tensor "
                            f"(got {t.dtype if torch.is_tensor(t) else type(t).__name__})")
        first = t if first is None else first
        if t.device != first.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the first input on {first.device}")


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------

_NORMS = ("none", "layer", "rms")
_GATES = ("none", "sigmoid", "silu")


def _eager_one_norm(x, kind, weight, bias, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * _wide(weight)
    return x if bias is None else x + _wide(bias)


def residual_norm(h, x=None, *, post="none", post_weight=None, post_bias=None, gate=None,
                  gate_act="silu", scale=None, pre="layer", pre_weight=None, pre_bias=None,
                  eps=1e-5):
    """A block's output norm, gate, residual scale and addition, and the next block's norm.

    ``p = post(h)``, ``u = p * act(gate)``, ``r = x + scale * u``, ``y = pre(r)``.

    Parameters
    ----------
    h : (..., D)
        What the block computed.
    x : (..., D), optional
        The residual stream; without it ``r = u`` and ``scale`` must be ``None``.
    post, pre : "none", "layer" or "rms"
        The norms over the last dimension, with ``post_weight``, ``post_bias``,
        ``pre_weight``, ``pre_bias`` (D), each optional.
    gate : broadcastable to ``h``, optional
        ``act`` is ``gate_act``, "sigmoid" or "silu".
    scale : (D) or float, optional

    Returns
    -------
    ``(r, y)``, or ``r`` alone if ``pre`` is "none", in the promoted type of ``h`` and ``x``.
    Norms and sums are in 32 bits or more; ``y`` is the norm of ``r`` before it is rounded.
    """
    vectors = dict(post_weight=post_weight, post_bias=post_bias, pre_weight=pre_weight,
                   pre_bias=pre_bias)
    number = 1.0
    if scale is not None and not torch.is_tensor(scale):
        scale, number = None, float(scale)
    _check_floats("residual_norm", h=h, x=x, gate=gate, scale=scale, **vectors)
    if post not in _NORMS or pre not in _NORMS:
        raise ValueError(f"residual_norm: post and pre are each one of {_NORMS} "
                         f"(got {post!r} and {pre!r})")
    if gate is None:
        gate_act = "none"
    elif gate_act not in _GATES[1:]:
        raise ValueError(f"residual_norm: gate_act is one of {_GATES[1:]} (got {gate_act!r})")
    if h.dim() == 0 or h.shape[-1] == 0:
        raise ValueError(f"residual_norm: h needs a last dimension (got shape {tuple(h.shape)})")
    if x is not None and x.shape != h.shape:
        raise ValueError(f"residual_norm: x has shape {tuple(x.shape)}, h {tuple(h.shape)}")
    if x is None and (scale is not None or number != 1.0):
        raise ValueError("residual_norm: scale scales the block's part of a sum, so it needs x")
    for name, t in (("scale", scale), *vectors.items()):
        if t is not None and t.shape != h.shape[-1:]:
            raise ValueError(f"residual_norm: {name} has shape {tuple(t.shape)}, not "
                             f"({h.shape[-1]},)")
    for kind, name in ((post, "post"), (pre, "pre")):
        if kind == "none" and not (vectors[name + "_weight"] is None
                                   and vectors[name + "_bias"] is None):
            raise ValueError(f"residual_norm: {name}_weight or {name}_bias without a {name} norm")
    if gate is not None and gate.shape != h.shape:
        gate = gate.expand_as(h)
    if h.numel():
        out = _dispatch("residual_norm", h.is_cuda, lambda backend: backend.residual_norm_impl(
            h, x, gate, scale, post_weight, post_bias, pre_weight, pre_bias, post, gate_act, pre,
            number, eps))
        if out is not None:
            return out
    dtype = h.dtype if x is None else torch.promote_types(h.dtype, x.dtype)
    u = _wide(h)
    if post != "none":
        u = _eager_one_norm(u, post, post_weight, post_bias, eps)
    if gate is not None:
        g = _wide(gate)
        u = u * (torch.sigmoid(g) if gate_act == "sigmoid" else torch.nn.functional.silu(g))
    if x is not None:
        u = _wide(x) + (number * u if scale is None else _wide(scale) * u)
    if pre == "none":
        return u.to(dtype)
    return u.to(dtype), _eager_one_norm(u, pre, pre_weight, pre_bias, eps).to(dtype)
