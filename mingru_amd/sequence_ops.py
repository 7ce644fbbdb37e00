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

__all__ = ["linear_attention", "linear_attention_step", "linear_cross_entropy", "residual_norm"]

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
        if not is_cuda:
            raise scans.ScanFallback("HIP kernels need GPU tensors")
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


# ---------------------------------------------------------------------------
# linear_attention
# ---------------------------------------------------------------------------

_EAGER_CHUNK = 64


def _over(g: torch.Tensor) -> torch.Tensor:
    """Steps whose factor is below the smallest normal float start over."""
    return g.double() * 1.4426950408889634 < -126.0


def _spans(total, count, lower):
    """``exp`` of the sums between two tokens, 0 where a step in between starts over."""
    diff = total[..., :, None] - total[..., None, :]
    keep = lower & (count[..., :, None] == count[..., None, :])
    return torch.exp(torch.where(keep, diff, torch.full_like(diff, -torch.inf)))


def _eager_linear_attention(q, k, v, g, h, lengths, scale):
    """Heads repeated, every input in the computing type; one chunk after another."""
    B, T, H, _ = q.shape
    if lengths is not None:
        live = torch.arange(T, device=q.device) < lengths[:, None].to(q.device)
        q, k, v = (torch.where(live[..., None, None], t, torch.zeros_like(t)) for t in (q, k, v))
        g = torch.where(live[..., None], g, torch.zeros_like(g))
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    g = g.transpose(1, 2)
    out = []
    for at in range(0, T, _EAGER_CHUNK):
        qc, kc, vc, gc = (t[:, :, at : at + _EAGER_CHUNK] for t in (q, k, v, g))
        over = _over(gc)
        count = over.cumsum(-1)
        total = torch.where(over, torch.zeros_like(gc), gc).double().cumsum(-1)
        lower = torch.ones(gc.shape[-1], gc.shape[-1], dtype=torch.bool, device=q.device).tril()
        D = _spans(total, count, lower).to(q.dtype)
        carried = torch.where(count == 0, total.exp(), torch.zeros_like(total)).to(q.dtype)
        # Past a start the state before is left out, in the gradients too, rather than multiplied
        # by 0, which would keep what is not finite.
        over = (count > 0)[..., None]
        through = (qc.masked_fill(over, 0) @ h).masked_fill(over, 0)
        o = carried[..., None] * through + ((qc @ kc.transpose(-1, -2)) * D) @ vc
        out.append(scale * o)
        h = (carried[..., -1, None, None] * h.masked_fill(over[..., -1, :, None], 0)
             + (kc * D[..., -1, :, None]).transpose(-1, -2) @ vc)
    return torch.cat(out, 2).transpose(1, 2), h


def _attention_checks(what, q, k, v, log_decay, h, lead):
    """Shared argument checks; ``lead``: the dimensions before the heads."""
    _check_floats(what, q=q, k=k, v=v, log_decay=log_decay, h=h)
    n = len(lead)
    if q.dim() != n + 2 or k.shape != q.shape or v.dim() != n + 2 or v.shape[:n] != q.shape[:n]:
        raise ValueError(
            f"{what}: q and k are {(*lead, 'Hk', 'dk')}, v is {(*lead, 'H', 'dv')} (got "
            f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)})")
    Hk, dk = q.shape[n:]
    H, dv = v.shape[n:]
    if Hk < 1 or H < 1 or H % Hk or dk < 1 or dv < 1:
        raise ValueError(f"{what}: the {H} heads of v are not a multiple of the {Hk} of q and k, "
                         "or a size is 0")
    if log_decay.shape != (*q.shape[:n], H) and log_decay.shape != (H,):
        raise ValueError(f"{what}: log_decay is {(*lead, 'H')} or (H,) (got "
                         f"{tuple(log_decay.shape)})")
    if h is not None and h.shape != (q.shape[0], H, dk, dv):
        raise ValueError(f"{what}: the state is (B, H, dk, dv) = {(q.shape[0], H, dk, dv)} (got "
                         f"{tuple(h.shape)})")


def _attention_types(q, k, v, log_decay, h):
    """Inputs in one type, decays and state in 32 bits (64 where an input has them)."""
    dtype = q.dtype
    if k.dtype is dtype and v.dtype is dtype and dtype is not torch.float64 and \
            log_decay.dtype is torch.float32 and (h is None or h.dtype is torch.float32):
        return q, k, v, log_decay, h
    dtype = torch.promote_types(torch.promote_types(dtype, k.dtype), v.dtype)
    wide = torch.float64 if torch.float64 in (dtype, log_decay.dtype) else torch.float32
    if wide == torch.float64:
        dtype = wide
    return (q.to(dtype), k.to(dtype), v.to(dtype), log_decay.to(wide),
            None if h is None else h.to(wide))


def linear_attention(q, k, v, log_decay, h_0=None, lengths=None, scale=None):
    """Attention through a state that decays: a prompt's or a training batch's whole pass.

    ``S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T`` and ``o_t = scale * S_t^T q_t`` for each
    sequence and head.  On the GPU the kernels take head sizes up to 128; larger ones run the
    eager body, with the warning of a decline.

    Parameters
    ----------
    q, k : (B, T, Hk, dk)
    v : (B, T, H, dv)
        ``Hk`` divides ``H``; each query and key head serves ``H / Hk`` heads in a row.
    log_decay : (B, T, H), or (H) for one decay a head
        At most 0.  ``-inf``, and any value whose factor is below the smallest normal float,
        starts a new document: nothing of the state before is seen after it, whatever it holds.
    h_0 : (B, H, dk, dv), optional
        The state to start from, 0 by default.
    lengths : (B) integers, optional
        Tokens of right-padded sequences.  The rest is not read; its outputs and gradients are
        0, and the final state is the one after a sequence's last token.
    scale : float, optional
        ``dk ** -0.5`` by default.

    Returns
    -------
    ``o`` (B, T, H, dv) in the inputs' type and the final state (B, H, dk, dv) in 32 bits (64
    for float64 inputs).  Differentiable in every floating input.
    """
    what = "linear_attention"
    _attention_checks(what, q, k, v, log_decay, h_0, ("B", "T"))
    if lengths is not None:
        if not torch.is_tensor(lengths) or lengths.dtype.is_floating_point or \
                lengths.dtype == torch.bool:
            raise TypeError(f"{what}: lengths must be a tensor of integers")
        if lengths.shape != q.shape[:1] or lengths.device != q.device:
            raise ValueError(f"{what}: lengths is (B,) on the inputs' device (got "
                             f"{tuple(lengths.shape)} on {lengths.device})")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v, log_decay, h_0 = _attention_types(q, k, v, log_decay, h_0)
    if q.numel() and v.numel():
        out = _dispatch(what, q.is_cuda, lambda backend: backend.linear_attention_impl(
            q, k, v, log_decay, h_0, lengths, scale))
        if out is not None:
            return out
    (B, T, Hk, dk), (H, dv) = q.shape, v.shape[2:]
    wide = log_decay.dtype
    h = q.new_zeros(B, H, dk, dv, dtype=wide) if h_0 is None else h_0
    if T == 0 or B == 0:
        return q.new_zeros(B, T, H, dv), h.clone()
    rep = H // Hk
    o, h = _eager_linear_attention(
        q.to(wide).repeat_interleave(rep, 2), k.to(wide).repeat_interleave(rep, 2), v.to(wide),
        log_decay.expand(B, T, H), h, lengths, scale)
    return o.to(q.dtype), h


@torch.no_grad()
def linear_attention_step(q_t, k_t, v_t, log_decay_t, h_prev=None, scale=None):
    """One token of :func:`linear_attention`: ``q_t``, ``k_t`` (B, Hk, dk), ``v_t`` (B, H, dv),
    ``log_decay_t`` (B, H) or (H), ``h_prev`` (B, H, dk, dv).  Returns ``o_t`` (B, H, dv) and the
    new state; no gradients."""
    what = "linear_attention_step"
    _attention_checks(what, q_t, k_t, v_t, log_decay_t, h_prev, ("B",))
    scale = q_t.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v, g, h = _attention_types(q_t, k_t, v_t, log_decay_t, h_prev)
    (B, Hk, dk), (H, dv) = q.shape, v.shape[1:]
    if h is None:
        h = torch.zeros(B, H, dk, dv, dtype=g.dtype, device=q.device)
    if B:
        out = _dispatch(what, q.is_cuda, lambda backend: backend.linear_attention_step_impl(
            q, k, v, g, h, scale))
        if out is not None:
            return out
    rep = H // Hk
    kw, qw = (t.to(g.dtype).repeat_interleave(rep, 1) for t in (k, q))
    # Selected, not multiplied by 0, which would keep what is not finite.
    kept = torch.where(_over(g).expand(B, H)[..., None, None], torch.zeros_like(h),
                       g.exp().expand(B, H)[..., None, None] * h)
    h = kept + kw[..., None] * v.to(g.dtype)[..., None, :]
    return (scale * (qw[..., None, :] @ h)[..., 0, :]).to(q.dtype), h


# ---------------------------------------------------------------------------
# linear_cross_entropy
# ---------------------------------------------------------------------------

_REDUCTIONS = ("none", "mean", "sum")


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index=-100, reduction="mean"):
    """Softmax cross entropy of ``x @ weight.T + bias`` against ``target``, without keeping the
    logits: on the GPU they are formed tile by tile, and again in the backward pass in pieces of
    the vocabulary.  There, with more than 128 rows, float32 weights are held to 2**-39 of their
    largest magnitude.

    Parameters
    ----------
    x : (..., D)
    weight : (V, D)
    target : (...) integers
        Rows with ``ignore_index`` are left out: they are not read, their losses and gradients
        are 0.  Any other value outside the vocabulary raises ``IndexError`` on the CPU; on the
        GPU, where looking would wait for it, that row's loss and all gradients that it is part
        of are NaN.
    bias : (V), optional
    reduction : "mean", "sum" or "none"
        "mean" is over the rows that count, 0 if there are none.

    Returns the loss in 32 bits (64 for float64 inputs): a scalar, or each row's in ``target``'s
    shape for "none".
    """
    what = "linear_cross_entropy"
    _check_floats(what, x=x, weight=weight, bias=bias)
    if not torch.is_tensor(target) or target.dtype.is_floating_point or \
            target.dtype in (torch.bool, torch.complex64, torch.complex128):
        raise TypeError(f"{what}: target must be a tensor of integers")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{what}: reduction is one of {_REDUCTIONS} (got {reduction!r})")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"{what}: x is (..., D) and weight (V, D) (got {tuple(x.shape)} and "
                         f"{tuple(weight.shape)})")
    if target.shape != x.shape[:-1] or target.device != x.device:
        raise ValueError(f"{what}: target has x's leading shape {tuple(x.shape[:-1])} and device "
                         f"(got {tuple(target.shape)} on {target.device})")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"{what}: bias is (V,) = ({weight.shape[0]},) (got {tuple(bias.shape)})")
    dtype = torch.promote_types(x.dtype, weight.dtype)
    if bias is not None:
        dtype = torch.promote_types(dtype, bias.dtype)
        bias = bias.to(dtype)
    x, weight = x.to(dtype), weight.to(dtype)
    if target.numel():
        out = _dispatch(what, x.is_cuda, lambda backend: backend.linear_cross_entropy_impl(
            x, weight, target, bias, ignore_index, reduction))
        if out is not None:
            return out
    t = target.reshape(-1)
    rows = torch.nonzero(t != ignore_index)[:, 0]
    at = t[rows].long()
    outside = (at < 0) | (at >= weight.shape[0])
    if bool(outside.any()):
        raise IndexError(f"{what}: target {int(at[outside][0])} is outside the vocabulary of "
                         f"{weight.shape[0]}")
    logits = _wide(x.reshape(-1, x.shape[-1])[rows]) @ _wide(weight).t()
    if bias is not None:
        logits = logits + _wide(bias)
    each = torch.logsumexp(logits, -1) - logits.gather(1, at[:, None])[:, 0]
    if reduction == "none":
        return each.new_zeros(t.shape).index_put((rows,), each).view(target.shape)
    return each.sum() / max(1, rows.numel()) if reduction == "mean" else each.sum()
