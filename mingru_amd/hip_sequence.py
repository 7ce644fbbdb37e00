"""HIP backend of :mod:`mingru_amd.sequence_ops`.

Same manners as :mod:`mingru_amd.hip_scans`: ``*_impl`` functions take the public
function's checked arguments, run on torch's current stream with outputs and workspaces
from torch's caching allocator, differentiate through ``torch.autograd.Function`` wrappers
(no double backward, no forward mode), and raise ``ScanFallback`` for a call they decline.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .hip_scans import (
    ScanFallback,
    _call,
    _funnel,
    _ptr,
    _size,
    _stream,
    _workspace,
    column_sums,
)

__all__ = [
    "linear_attention_impl",
    "linear_attention_step_impl",
    "linear_cross_entropy_impl",
    "residual_norm_impl",
]

_DTYPE_TAG = {torch.float32: 0, torch.bfloat16: 1}


def _half_to_float(*ts):
    """fp16 inputs run the fp32 kernels on upcast copies; float64 declines."""
    out = []
    for t in ts:
        if t is not None and t.dtype not in _DTYPE_TAG:
            if t.dtype != torch.float16:
                raise ScanFallback(f"the kernels compute in fp32; {t.dtype} stays on the eager path")
            t = t.float()
        out.append(t)
    return out


def _no_tangents(what, *ts):
    """Declines inputs with a forward-mode tangent: the native calls read the primals alone, and
    an output without a tangent counts as a constant."""
    # Outside of every dual level (-1), where nothing has a tangent, nothing is looked at.
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise ScanFallback(f"{what} kernels have no forward-mode derivatives")


# ---------------------------------------------------------------------------
# residual_norm
# ---------------------------------------------------------------------------

_NORM_MAX_D = 8192
_NORM_TAG = {"none": 0, "layer": 1, "rms": 2}
_GATE_TAG = {"none": 0, "sigmoid": 1, "silu": 2}


def _rows(t, D):
    """``t`` as rows of ``D`` consecutive elements and the elements between them."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, D
    if t.stride(-1) != 1 and D > 1:
        t = t.contiguous()
    t = t.reshape(-1, D)
    if t.shape[0] == 1:
        return t, D
    if t.stride(0) < D:
        t = t.contiguous()
    return t, t.stride(0)


def _residual_norm_fwd(h, x, gate, vectors, kinds, number, eps, keep):
    """``r``, ``y`` or ``None``, and for the backward (``keep``) the rows' statistics and the tags."""
    D = h.shape[-1]
    h2, ldh = _rows(h, D)
    x2, ldx = _rows(x, D)
    g2, ldg = _rows(gate, D)
    rows = h.numel() // D
    r = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    y = torch.empty_like(r) if kinds[2] else None
    stats = None
    if keep and (kinds[0] or kinds[2]):
        stats = torch.empty(rows, 4, dtype=torch.float32, device=h.device)
    first = next((t for t in vectors if t is not None), h)
    tags = (_DTYPE_TAG[h.dtype], _DTYPE_TAG[first.dtype], *kinds)
    scale, post_w, post_b, pre_w, pre_b = vectors
    _call("mg_residual_norm_fwd", *tags, _ptr(h2), ldh, _ptr(x2), ldx, _ptr(g2), ldg,
          _ptr(scale), number, _ptr(post_w), _ptr(post_b), _ptr(pre_w), _ptr(pre_b), _ptr(r),
          _ptr(y), _ptr(stats), rows, D, eps, _stream(h))
    return r, y, stats, tags


def _grad_wanted(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


class _ResidualNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, x, gate, scale, post_w, post_b, pre_w, pre_b, kinds, number, eps):
        ctx.set_materialize_grads(False)
        vectors = [t if t is None else t.contiguous()
                   for t in (scale, post_w, post_b, pre_w, pre_b)]
        r, y, stats, ctx.tags = _residual_norm_fwd(h, x, gate, vectors, kinds, number, eps, True)
        ctx.save_for_backward(h, x, gate, stats, *vectors)
        ctx.number, ctx.eps = number, eps
        return r if y is None else (r, y)

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dy=None):
        h, x, gate, stats, scale, post_w, post_b, pre_w, pre_b = ctx.saved_tensors
        D, dev = h.shape[-1], h.device
        if dr is None and dy is None:
            return (None,) * 11
        need = ctx.needs_input_grad
        post, act, _ = ctx.tags[2:]
        h2, ldh = _rows(h, D)
        x2, ldx = _rows(x, D)
        g2, ldg = _rows(gate, D)
        dr2, lddr = _rows(dr, D)
        dy2, lddy = _rows(dy, D)
        rows = h.numel() // D

        def like(i):
            return torch.empty(h.shape, dtype=h.dtype, device=dev) if need[i] else None

        # The block's part of a plain sum has the stream's own gradient.
        same = bool(need[1]) and not (post or act) and scale is None and ctx.number == 1.0
        dx, dgate = like(1), like(2)
        dh = None if same else like(0)
        vectors = [torch.empty(D, dtype=t.dtype, device=dev) if need[3 + i] else None
                   for i, t in enumerate((scale, post_w, post_b, pre_w, pre_b))]
        ws = None
        if any(v is not None for v in vectors):
            ws = _workspace(_size("mg_residual_norm_workspace_bytes", rows, D), dev)
        _call("mg_residual_norm_bwd", *ctx.tags, _ptr(h2), ldh, _ptr(x2), ldx, _ptr(g2), ldg,
              _ptr(scale), ctx.number, _ptr(post_w), _ptr(post_b), _ptr(pre_w), _ptr(stats),
              _ptr(dr2), lddr, _ptr(dy2), lddy, _ptr(dh), _ptr(dx), _ptr(dgate),
              *[_ptr(v) for v in vectors], rows, D, ctx.eps, _ptr(ws),
              0 if ws is None else ws.numel(),
              _stream(h))
        return (dx if same and need[0] else dh, dx, dgate, *vectors, None, None, None)


def residual_norm_impl(h, x, gate, scale, post_w, post_b, pre_w, pre_b, post, act, pre, number,
                       eps):
    """``residual_norm`` on checked arguments (``number``: the scale where ``scale`` is None)."""
    _no_tangents("residual_norm", h, x, gate, scale, post_w, post_b, pre_w, pre_b)
    if h.shape[-1] > _NORM_MAX_D:
        raise ScanFallback(f"residual_norm kernels hold rows of at most {_NORM_MAX_D} elements "
                           f"(got {h.shape[-1]})")
    dtype = h.dtype if x is None else torch.promote_types(h.dtype, x.dtype)
    h, x, gate, *vectors = _half_to_float(h, x, gate, scale, post_w, post_b, pre_w, pre_b)
    if any(t is not None and t.dtype != h.dtype for t in (x, gate)):
        h, x, gate = (t if t is None else t.float() for t in (h, x, gate))
    if any(t is not None and t.dtype != torch.bfloat16 for t in vectors) or \
            h.dtype == torch.float32:
        vectors = [t if t is None else t.float() for t in vectors]
    kinds = (_NORM_TAG[post], _GATE_TAG[act], _NORM_TAG[pre])
    if _grad_wanted(h, x, gate, *vectors):
        out = _funnel("residual_norm", _ResidualNormFn.apply, h, x, gate, *vectors, kinds, number,
                      float(eps))
    else:
        vectors = [t if t is None else t.contiguous() for t in vectors]
        r, y, *_ = _funnel("residual_norm", _residual_norm_fwd, h, x, gate, vectors, kinds, number,
                           float(eps), False)
        out = r if y is None else (r, y)
    if h.dtype == dtype:
        return out
    return tuple(t.to(dtype) for t in out) if kinds[2] else out.to(dtype)


# ---------------------------------------------------------------------------
# linear_attention
# ---------------------------------------------------------------------------

_ATTENTION_MAX_D = 128
_STEP_PAIRS = 2**24  # of a sequence and a head; the pass has its limits from the C entry


def _last_dense(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _decay_strides(g, n):
    """Strides of ``g`` over ``n`` leading dimensions and the heads; a decay for each head has none."""
    return (0,) * n + (g.stride(0),) if g.dim() == 1 else g.stride()


def _array(values):
    return (ctypes.c_int64 * len(values))(*values)


def _linear_attention_fwd(q, k, v, g, h0, lengths, scale):
    """``o``, the final state, what the backward needs of the pass, sizes and strides."""
    (B, T, Hk, dk), (H, dv) = q.shape, v.shape[2:]
    tag, dev = _DTYPE_TAG[q.dtype], q.device
    size = (tag, B, T, H, Hk, dk, dv)
    o = torch.empty(B, T, H, dv, dtype=q.dtype, device=dev)
    h = torch.empty(B, H, dk, dv, dtype=torch.float32, device=dev)
    state = _workspace(_size("mg_linear_attention_state_bytes", *size), dev)
    strides = (*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *_decay_strides(g, 2))
    _call("mg_linear_attention_fwd", tag, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _array(strides),
          _ptr(lengths), _ptr(h0), _ptr(o), _ptr(h), _ptr(state), state.numel(), B, T, H, Hk,
          dk, dv, scale, _stream(q))
    return o, h, state, size, strides


class _LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, h0, lengths, scale):
        ctx.set_materialize_grads(False)
        q, k, v = (_last_dense(t) for t in (q, k, v))
        o, h, state, ctx.size, ctx.strides = _linear_attention_fwd(q, k, v, g, h0, lengths, scale)
        ctx.save_for_backward(q, k, v, g, h0, lengths, h, state)
        ctx.scale = scale
        return o, h

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dh):
        if do is None and dh is None:
            return (None,) * 7
        q, k, v, g, h0, lengths, h, state = ctx.saved_tensors
        tag, B, T, H, Hk, dk, dv = ctx.size
        dev = q.device
        if do is None:
            do = torch.zeros(B, T, H, dv, dtype=q.dtype, device=dev)
        do = _last_dense(do)
        if dh is not None:
            dh = dh.contiguous()
        dq, dk_, dv_ = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        dg = torch.empty(B, T, H, dtype=torch.float32, device=dev)
        dh0 = torch.empty_like(h) if ctx.needs_input_grad[4] else None
        ws = _workspace(_size("mg_linear_attention_workspace_bytes", *ctx.size), dev)
        _call("mg_linear_attention_bwd", tag, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(do),
              _array((*ctx.strides, *do.stride()[:3])), _ptr(lengths), _ptr(h0), _ptr(h),
              _ptr(state), _ptr(dh), _ptr(dq), _ptr(dk_), _ptr(dv_), _ptr(dg), _ptr(dh0), B, T, H,
              Hk, dk, dv, ctx.scale, _ptr(ws), ws.numel(), _stream(q))
        if g.dim() == 1 and ctx.needs_input_grad[3]:
            dg = column_sums(dg.view(B * T, H))
        return dq, dk_, dv_, dg, dh0, None, None


def linear_attention_impl(q, k, v, g, h0, lengths, scale):
    """``linear_attention`` on checked arguments of one type."""
    _no_tangents("linear_attention", q, k, v, g, h0)
    if max(q.shape[-1], v.shape[-1]) > _ATTENTION_MAX_D:
        raise ScanFallback(f"linear_attention kernels take head sizes up to {_ATTENTION_MAX_D} "
                           f"(got {q.shape[-1]} and {v.shape[-1]})")
    dtype = q.dtype
    q, k, v, g, h0 = _half_to_float(q, k, v, g, h0)
    (B, T, Hk, dk), (H, dv) = q.shape, v.shape[2:]
    if not _size("mg_linear_attention_state_bytes", _DTYPE_TAG[q.dtype], B, T, H, Hk, dk, dv):
        raise ScanFallback(f"linear_attention kernels take fewer than 2^23 pairs of a sequence and a "
                           f"head, up to 2^16 heads and 2^32 tokens (got {B} x {H} and {T})")
    if h0 is not None:
        h0 = h0.contiguous()
    if lengths is not None:
        if T >= 2**31:
            raise ScanFallback(f"linear_attention kernels take lengths below 2^31 (got {T} tokens)")
        if lengths.dtype.itemsize > 4 or lengths.dtype == torch.uint32:
            # The type to come holds what matters of them only.
            lengths = lengths.to(torch.int64).clamp(0, T)
        lengths = lengths.to(torch.int32).contiguous()
    if _grad_wanted(q, k, v, g, h0):
        o, h = _funnel("linear_attention", _LinearAttentionFn.apply, q, k, v, g, h0, lengths, scale)
    else:
        q, k, v = (_last_dense(t) for t in (q, k, v))
        o, h, *_ = _funnel("linear_attention", _linear_attention_fwd, q, k, v, g, h0, lengths,
                           scale)
    return o if o.dtype == dtype else o.to(dtype), h


def linear_attention_step_impl(q, k, v, g, h, scale):
    """``linear_attention_step`` on checked arguments of one type."""
    _no_tangents("linear_attention_step", q, k, v, g, h)
    (B, Hk, dk), (H, dv) = q.shape, v.shape[1:]
    if B * H >= _STEP_PAIRS:
        raise ScanFallback(f"linear_attention_step kernels take fewer than 2^24 pairs of a sequence "
                           f"and a head (got {B} x {H})")
    dtype = q.dtype
    q, k, v, g, h = _half_to_float(q, k, v, g, h)
    q, k, v = (_last_dense(t) for t in (q, k, v))
    h = h.contiguous()
    o = torch.empty(B, H, dv, dtype=q.dtype, device=q.device)
    h_out = torch.empty_like(h)
    strides = (*q.stride()[:2], *k.stride()[:2], *v.stride()[:2], *_decay_strides(g, 1))
    _funnel("linear_attention_step", _call, "mg_linear_attention_step", _DTYPE_TAG[q.dtype],
            _ptr(q), _ptr(k), _ptr(v), _ptr(g), _array(strides), _ptr(h), _ptr(o), _ptr(h_out), B,
            H, Hk, dk, dv, scale, _stream(q))
    return o if o.dtype == dtype else o.to(dtype), h_out


# ---------------------------------------------------------------------------
# linear_cross_entropy
# ---------------------------------------------------------------------------

_REDUCTION_TAG = {"none": 0, "mean": 1, "sum": 2}


def _vocab_loss_fwd(x, w, bias, target, ignore_index, reduction):
    """The loss, what the backward needs of the pass, and sizes; ``w`` dense and aligned."""
    x2, ldx = _rows(x, x.shape[-1])
    N, (V, D) = target.numel(), w.shape
    tag, dev = _DTYPE_TAG[x.dtype], x.device
    state = _workspace(_size("mg_vocab_loss_state_bytes", tag, N, V, D), dev)
    ws = _workspace(_size("mg_vocab_loss_fwd_workspace_bytes", tag, N, V, D), dev)
    loss = torch.empty(N if reduction == 0 else (), dtype=torch.float32, device=dev)
    _call("mg_vocab_loss_fwd", tag, _ptr(x2), ldx, _ptr(w), _ptr(bias), _ptr(target),
          ignore_index, reduction, _ptr(loss), N, V, D, _ptr(state), state.numel(), _ptr(ws),
          ws.numel(), _stream(x))
    return loss, state, (tag, N, V, D)


def _dense_aligned(w):
    w = w.contiguous()
    return w.clone() if w.data_ptr() % 16 else w


class _VocabLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, target, ignore_index, reduction):
        w, bias = _dense_aligned(w), bias if bias is None else bias.contiguous()
        loss, state, ctx.size = _vocab_loss_fwd(x, w, bias, target, ignore_index, reduction)
        ctx.save_for_backward(w, bias, state)
        ctx.shape, ctx.reduction = x.shape, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        w, bias, state = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = torch.empty(ctx.shape, dtype=w.dtype, device=w.device) if need[0] else None
        db = torch.empty_like(bias) if need[2] else None
        dw = torch.empty_like(w) if need[1] or db is not None else None
        nbytes = _size("mg_vocab_loss_bwd_workspace_bytes", *ctx.size)
        if dx is None:
            nbytes -= _size("mg_vocab_loss_bwd_dx_bytes", *ctx.size)
        ws = _workspace(nbytes, w.device)
        tag, N, V, D = ctx.size
        _call("mg_vocab_loss_bwd", tag, _ptr(w), _ptr(bias), _ptr(dloss.contiguous()),
              ctx.reduction, _ptr(dx), _ptr(dw), _ptr(db), N, V, D, _ptr(state), _ptr(ws),
              ws.numel(), _stream(w))
        return dx, dw if need[1] else None, db, None, None, None


def linear_cross_entropy_impl(x, weight, target, bias, ignore_index, reduction):
    """``linear_cross_entropy`` on checked arguments of one type."""
    _no_tangents("linear_cross_entropy", x, weight, bias)
    x, weight, bias = _half_to_float(x, weight, bias)
    N, (V, D) = target.numel(), weight.shape
    if not _size("mg_vocab_loss_state_bytes", _DTYPE_TAG[x.dtype], N, V, D):
        raise ScanFallback(f"linear_cross_entropy kernels take fewer than 2^30 rows and "
                           f"vocabulary entries and rows of at most 2^20 (got {N}, {V}, {D})")
    t = target.reshape(-1).to(torch.int64).contiguous()
    rest = t, int(ignore_index), _REDUCTION_TAG[reduction]
    if _grad_wanted(x, weight, bias):
        loss = _funnel("linear_cross_entropy", _VocabLossFn.apply, x, weight, bias, *rest)
    else:
        loss = _funnel("linear_cross_entropy", _vocab_loss_fwd, x, _dense_aligned(weight),
                       bias if bias is None else bias.contiguous(), *rest)[0]
    return loss.view(target.shape) if reduction == "none" else loss
