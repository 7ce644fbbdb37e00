"""HIP backend of :mod:`mingru_amd.decode_ops`.

Same manners as :mod:`mingru_amd.hip_sequence`: ``*_impl`` functions take the public
function's checked arguments, run on torch's current stream with outputs and workspaces from
torch's caching allocator, and raise ``ScanFallback`` for a call they decline.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .hip_scans import ScanFallback, _call, _funnel, _ptr, _size, _stream, _workspace
from .hip_sequence import _array, _last_dense, _no_tangents

__all__ = [
    "beam_select_impl",
    "paged_attention_step_impl",
    "paged_cache_append_impl",
    "reorder_states_impl",
]

_DTYPE_TAG = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _tag(what, t) -> int:
    tag = _DTYPE_TAG.get(t.dtype)
    if tag is None:
        raise ScanFallback(f"{what} kernels take float32, bfloat16 and float16 (got {t.dtype})")
    return tag


def _launch(what, t, name, *args):
    """``name`` of the C ABI on ``t``'s device, whose default stream is another device's otherwise."""
    if torch.cuda.current_device() != t.device.index:
        with torch.cuda.device(t.device):
            return _funnel(what, _call, name, *args, _stream(t))
    return _funnel(what, _call, name, *args, _stream(t))


def _ints(*ts):
    """The tensors as int32 or int64 with a dense last dimension, and which are the latter."""
    wide, out = 0, []
    for i, t in enumerate(ts):
        if t is not None:
            if t.dtype is not torch.int32:
                t = t.to(torch.int64)
                wide |= 1 << i
            t = _last_dense(t)
        out.append(t)
    return (wide, *out)


def _cache(what, name, t):
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ScanFallback(f"{what} kernels need {name}'s last dimension dense")
    return t


def paged_cache_append_impl(k, v, k_cache, v_cache, pages, start, q, lengths, frequencies,
                            interleaved):
    """``paged_cache_append`` on checked arguments; a tuple of the rotated queries or ``None``."""
    what = "paged_cache_append"
    _no_tangents(what, k, v, k_cache, v_cache, q, frequencies)
    tag = _tag(what, k)
    (B, T, Hk, dk), (N, _, P, dv) = k.shape, v_cache.shape
    _cache(what, "k_cache", k_cache), _cache(what, "v_cache", v_cache)
    if not (N and pages.shape[1]):
        # No token has a place: every page from 0 on is 1 of a cache of one, which nothing is written to.
        if q is None:
            return (None,)
        k_cache, v_cache = (c.new_empty(1, *c.shape[1:]) for c in (k_cache, v_cache))
        N, pages = 1, (torch.where(pages.long() < 0, -1, 1) if pages.shape[1]
                       else pages.new_ones(B, 1, dtype=torch.int64))
    H = 0 if q is None else q.shape[2]
    n = 0 if frequencies is None else frequencies.shape[0]
    if N >= 2**31 or P >= 2**31 or Hk * (dk + dv) + H * dk >= 2**26 or n > 1024:
        raise ScanFallback(f"{what} kernels take tokens of fewer than 2^26 elements, up to 1024 "
                           f"frequencies and fewer than 2^31 pages (got {N} of {P} tokens)")
    k, v = _last_dense(k), _last_dense(v)
    out, turned, qs = None, 0, (0, 0, 0)
    if q is not None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q = _last_dense(q)
        turned, qs = out.data_ptr(), q.stride()[:3]
    wide, pages, start, lengths = _ints(pages, start, lengths)
    if n:
        if frequencies.dtype not in (torch.float32, torch.float64):
            frequencies = frequencies.float()
        frequencies = frequencies.contiguous()
    strides = (*qs, *k.stride()[:3], *v.stride()[:3], *k_cache.stride()[:3], *v_cache.stride()[:3],
               pages.stride(0))
    _launch(what, k, "mg_paged_append", tag, _ptr(q) if H else 0, k.data_ptr(), v.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), turned, _array(strides), wide,
            pages.data_ptr(), start.data_ptr(), _ptr(lengths),
            int(n > 0 and frequencies.dtype is torch.float64), _ptr(frequencies), n,
            int(bool(interleaved)), B, T, H, Hk, dk, dv, N, pages.shape[1], P)
    # As torch's own writes do, for what autograd may have saved.
    increment_version([c for c in (k_cache, v_cache) if not c.is_inference()])
    return (out,)


def paged_attention_step_impl(q, k_cache, v_cache, pages, lengths, scale, window):
    """``paged_attention_step`` on checked arguments."""
    what = "paged_attention_step"
    _no_tangents(what, q, k_cache, v_cache)
    tag = _tag(what, q)
    (B, H, dk), (N, Hk, P, dv) = q.shape, v_cache.shape
    M = pages.shape[1]
    if not (N and M):  # no token has a place
        lost = torch.where(lengths.long() > 0, torch.nan, 0.0).to(q.dtype)
        return lost[:, None, None].expand(B, H, dv).contiguous()
    _cache(what, "k_cache", k_cache), _cache(what, "v_cache", v_cache)
    nbytes = _size("mg_paged_attention_workspace_bytes", tag, B, H, Hk, dk, dv, M, P)
    if not nbytes or N >= 2**31:
        raise ScanFallback(f"{what} kernels take head sizes up to 256, fewer than 2^24 heads of all "
                           f"sequences, tables of fewer than 2^31 - 1024 tokens and fewer than 2^31 "
                           f"pages (got {dk} and {dv}, {B} x {H}, {M} x {P} and {N})")
    q = _last_dense(q)
    size = q.element_size()
    row = 16 if dk * size % 16 == 0 else 8
    if dk * size % row == 0 and (q.data_ptr() | (q.stride(0) | q.stride(1)) * size) % row:
        # Small, and the kernels load the caches by vectors only together with the queries.
        q = q.clone(memory_format=torch.contiguous_format)
    wide, pages, lengths = _ints(pages, lengths)
    o = torch.empty(B, H, dv, dtype=q.dtype, device=q.device)
    ws = _workspace(nbytes, q.device)
    strides = (*q.stride()[:2], *k_cache.stride()[:3], *v_cache.stride()[:3], pages.stride(0))
    # A window that no sequence outgrows is none.
    window = 0 if window is None or window >= M * P else window
    _launch(what, q, "mg_paged_attention_step", tag, _ptr(q), _ptr(k_cache), _ptr(v_cache),
            _array(strides), wide, _ptr(pages), _ptr(lengths), _ptr(o), B, H, Hk, dk, dv, N, M, P,
            window, scale, _ptr(ws), ws.numel())
    return o


_BEAM_MAX_WIDTH = 64


def beam_select_impl(logits, scores, width, end, finished):
    """``beam_select`` on checked arguments."""
    what = "beam_select"
    _no_tangents(what, logits, scores)
    if scores.dtype == torch.float64:
        raise ScanFallback(f"{what} kernels take scores in 32 bits")
    tag = _tag(what, logits)
    B, K, V = logits.shape
    nbytes = _size("mg_beam_select_workspace_bytes", tag, B, K, V, width) \
        if width <= _BEAM_MAX_WIDTH else 0
    if not nbytes:
        raise ScanFallback(f"{what} kernels keep up to {_BEAM_MAX_WIDTH} of up to 256 beams, of fewer "
                           f"than 2^22 in all and 2^31 candidates a search (got {width} of {B} x {K} "
                           f"x {V})")
    logits, scores = _last_dense(logits), scores.float()
    dev = logits.device
    out = torch.empty(B, width, dtype=torch.float32, device=dev)
    parents, tokens = (torch.empty(B, width, dtype=torch.int64, device=dev) for _ in range(2))
    done = None if end is None else torch.empty(B, width, dtype=torch.bool, device=dev)
    ws = _workspace(nbytes, dev)
    strides = (*logits.stride()[:2], *scores.stride(),
               *((0, 0) if finished is None else finished.stride()))
    _launch(what, logits, "mg_beam_select", tag, _ptr(logits), _ptr(scores), _ptr(finished),
            _array(strides), -1 if end is None else int(end), _ptr(out), _ptr(parents),
            _ptr(tokens), _ptr(done), B, K, V, width, _ptr(ws), ws.numel())
    return (out, parents, tokens) if done is None else (out, parents, tokens, done)


def reorder_states_impl(tensors, parents, K):
    """``reorder_states`` on checked arguments: a list of tensors, of ``K`` rows a search."""
    what = "reorder_states"
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _no_tangents(what, *[t for t in tensors if t.dtype.is_floating_point])
    B, W = parents.shape
    if K == 0:  # no parent is one of them
        return [t.new_zeros(B * W, *t.shape[1:]) for t in tensors]
    if B * W >= 2**31 or K >= 2**31:
        raise ScanFallback(f"{what} kernels write fewer than 2^31 rows (got {B} x {W})")
    if parents.dtype not in (torch.int32, torch.int64):
        parents = parents.to(torch.int64)
    out, src, dst, strides, sizes, kept = [], [], [], [], [], []
    rows, same = B * K, W == K
    for t in tensors:
        if t.is_conj() or t.is_neg():
            t = t.resolve_conj().resolve_neg()
            kept.append(t)  # until the launch
        dense = t.is_contiguous()
        if dense and same:
            new = torch.empty_like(t)
        else:
            new = torch.empty((B * W, *t.shape[1:]), dtype=t.dtype, device=t.device)
        out.append(new)
        size = stride = t.nbytes // rows
        if size == 0:
            continue
        if not dense:
            if t[0].is_contiguous():
                stride = t.stride(0) * t.element_size()
            else:
                t = t.contiguous()
            kept.append(t)  # until the launch
        src.append(t.data_ptr())
        dst.append(new.data_ptr())
        strides.append(stride)
        sizes.append(size)
    if src:
        n = len(src)
        pointers, longs = ctypes.c_void_p * n, ctypes.c_int64 * n
        _launch(what, parents, "mg_reorder_rows", n, pointers(*src), pointers(*dst),
                longs(*strides), longs(*sizes), int(parents.dtype == torch.int64), _ptr(parents),
                *parents.stride(), B, K, W)
    return out
