"""Operators with which a language model answers: a paged cache of keys and values with the
attention that reads it, and a beam search's selection with the reordering of states.

The reference has none of them; its decoding is the mixers' ``step``
(``src/mingru/min_gru.py:1399-1448``).  They follow the contract of
:mod:`mingru_amd.sequence_ops`: ``MINGRU_SCAN`` picks the path on every call, GPU tensors run
the HIP kernels of :mod:`mingru_amd.hip_decode`, a decline falls back to the eager body with a
once-per-process warning (``auto``) or raises ``RuntimeError`` (``hip``), and CPU tensors run
the eager body, which defines the results.  None of them has gradients.

A paged cache is two tensors, keys (N, Hk, P, dk) and values (N, Hk, P, dv): N pages of P
tokens.  A sequence's token ``p`` lies in page ``pages[b, p // P]`` at ``p % P``.  Other orders
of the same dimensions are views of one (a cache (N, P, Hk, d) goes in as
``cache.transpose(1, 2)``).  Beams may share pages that none of them writes any more; with pages
of one token that is all but the newest, so such beams follow their parents by
``reorder_states`` of the page tables alone.
"""

from __future__ import annotations

import copy

import torch

from .sequence_ops import _check_floats, _dispatch, _wide

__all__ = ["beam_select", "paged_attention_step", "paged_cache_append", "reorder_states"]


_INTEGERS = {torch.int8, torch.int16, torch.int32, torch.int64, torch.uint8, torch.uint16,
             torch.uint32, torch.uint64}


def _check_whole(what: str, device, **tensors) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.dtype not in _INTEGERS:
            raise TypeError(f"{what}: {name} must be a tensor of integers (got "
                            f"{t.dtype if torch.is_tensor(t) else type(t).__name__})")
        if t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, the first input on {device}")


def _check_cache(what: str, k_cache, v_cache, pages, B: int) -> tuple:
    """N, Hk, P, dk and dv of the caches."""
    ks, vs, table = k_cache.shape, v_cache.shape, pages.shape
    if len(ks) != 4 or len(vs) != 4 or (ks[0], ks[1], ks[2]) != (vs[0], vs[1], vs[2]):
        raise ValueError(f"{what}: k_cache is (N, Hk, P, dk) and v_cache (N, Hk, P, dv) (got "
                         f"{tuple(ks)} and {tuple(vs)})")
    N, Hk, P, dk = ks
    if not (Hk and P and dk and vs[3]):
        raise ValueError(f"{what}: a size of the caches is 0 (got {tuple(ks)} and {tuple(vs)})")
    if len(table) != 2 or table[0] != B:
        raise ValueError(f"{what}: pages is (B, M) with B = {B} (got {tuple(table)})")
    return N, Hk, P, dk, vs[3]


def _check_one_type(what: str, **tensors) -> None:
    """Floating-point tensors of one type on one device."""
    dtype = device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a floating-point tensor (got "
                            f"{type(t).__name__})")
        if dtype is None:
            first, dtype, device = name, t.dtype, t.device
            if not dtype.is_floating_point:
                raise TypeError(f"{what}: {name} must be a floating-point tensor (got {dtype})")
        elif t.dtype is not dtype:
            raise TypeError(f"{what}: {name} has {first}'s type (got {t.dtype} and {dtype})")
        elif t.device != device:
            raise ValueError(f"{what}: {name} is on {t.device}, the first input on {device}")


# ---------------------------------------------------------------------------
# paged_cache_append
# ---------------------------------------------------------------------------


def _turned(x, position, frequencies, interleaved):
    """``x`` (B, T, heads, d) rotated by ``position`` (B, T)."""
    n = frequencies.numel()
    angle = position.double()[..., None] * frequencies.double()
    x = _wide(x)
    cos, sin = (f(angle).to(x.dtype)[:, :, None] for f in (torch.cos, torch.sin))
    part, rest = x[..., : 2 * n], x[..., 2 * n :]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((part, rest), -1)


def paged_cache_append(k, v, k_cache, v_cache, pages, start, *, q=None, lengths=None,
                       frequencies=None, interleaved=False):
    """Puts new tokens' keys and values into a paged cache, in place, with keys and queries
    rotated by their positions on the way.

    Token ``t`` of sequence ``b`` has position ``p = start[b] + t``.  With ``frequencies`` f,
    elements ``x_i`` and ``x_{i+n}`` (n frequencies; ``x_{2i}`` and ``x_{2i+1}`` if
    ``interleaved``) of each key and query become ``x_i cos(p f_i) - x_{i+n} sin(p f_i)`` and
    ``x_{i+n} cos(p f_i) + x_i sin(p f_i)``; angles are in 64 bits.  Elements from 2n on stay.
    Nothing of it has gradients: not the queries, nor what lies in the caches.

    Parameters
    ----------
    k : (B, T, Hk, dk)
    v : (B, T, Hk, dv)
    k_cache : (N, Hk, P, dk)
    v_cache : (N, Hk, P, dv)
        Written in place, at the new tokens alone.  One type for all of them and ``q``.
    pages : (B, M) integers
        A token whose page is negative is not kept.  No two tokens may have one place.
    start : (B) integers
        Tokens that each sequence has in the cache already.
    q : (B, T, H, dk), optional
    lengths : (B) integers, optional
        New tokens of right-padded sequences.  The rest is not read, and its queries are 0.
    frequencies : (n), optional
        Radians a position, up to half of ``dk`` of them; without, nothing is rotated.

    Returns
    -------
    The rotated ``q``, or ``None`` without one.  A token that lies behind its row of ``pages``,
    or whose page is not in the cache, raises ``IndexError`` in the eager body, on either device;
    with the kernels, where looking would wait for the GPU, it is not kept and its queries are NaN.
    """
    what = "paged_cache_append"
    _check_one_type(what, k=k, v=v, k_cache=k_cache, v_cache=v_cache, q=q)
    _check_whole(what, k.device, pages=pages, start=start, lengths=lengths)
    shape, vs = k.shape, v.shape
    if len(shape) != 4 or len(vs) != 4 or (shape[0], shape[1], shape[2]) != (vs[0], vs[1], vs[2]):
        raise ValueError(f"{what}: k is (B, T, Hk, dk) and v (B, T, Hk, dv) (got "
                         f"{tuple(shape)} and {tuple(vs)})")
    B, T, Hk, dk = shape
    N, heads, P, *sizes = _check_cache(what, k_cache, v_cache, pages, B)
    if heads != Hk or sizes != [dk, vs[3]]:
        raise ValueError(f"{what}: the caches hold {heads} heads of sizes {sizes}, k and v are "
                         f"{tuple(shape)} and {tuple(vs)}")
    if q is not None:
        qs = q.shape
        if len(qs) != 4 or qs[0] != B or qs[1] != T or qs[3] != dk:
            raise ValueError(f"{what}: q is (B, T, H, dk) = ({B}, {T}, H, {dk}) (got {tuple(qs)})")
    for name, t in (("start", start), ("lengths", lengths)):
        if t is not None and t.shape != (B,):
            raise ValueError(f"{what}: {name} is (B,) = ({B},) (got {tuple(t.shape)})")
    if frequencies is not None:
        _check_floats(what, k=k, frequencies=frequencies)
        n = frequencies.shape
        if len(n) != 1 or not 1 <= n[0] <= dk // 2:
            raise ValueError(f"{what}: frequencies is (n,) with n from 1 to dk / 2 = {dk // 2} (got "
                             f"{tuple(n)})")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise ValueError(f"{what}: {name} is written, so it must not be an expanded view")
    if B * T:
        done = _dispatch(what, k.is_cuda, lambda backend: backend.paged_cache_append_impl(
            k, v, k_cache, v_cache, pages, start, q, lengths, frequencies, interleaved),
            "hip_decode")
        if done is not None:
            return done[0]
    return _eager_append(k, v, k_cache, v_cache, pages, start, q, lengths, frequencies, interleaved)


@torch.no_grad()
def _eager_append(k, v, k_cache, v_cache, pages, start, q, lengths, frequencies, interleaved):
    what = "paged_cache_append"
    (B, T), (N, _, P, _) = k.shape[:2], k_cache.shape
    t = torch.arange(T, device=k.device)
    position = start.long()[:, None] + t
    live = (t < lengths.long()[:, None]) if lengths is not None else torch.ones_like(position) > 0
    b, t = torch.nonzero(live, as_tuple=True)
    at = position[b, t]
    if bool(((at < 0) | (at >= pages.shape[1] * P)).any()):
        raise IndexError(f"{what}: a token lies outside of its sequence's {pages.shape[1]} pages")
    page = pages.long()[b, at // P]
    if bool((page >= N).any()):
        raise IndexError(f"{what}: page {int(page.max())} is outside of the cache of {N}")
    kept = page >= 0
    b, t, at, page = b[kept], t[kept], at[kept], page[kept]
    turned = k if frequencies is None else _turned(k, position, frequencies, interleaved)
    k_cache[page, :, at % P] = turned[b, t].to(k_cache.dtype)
    v_cache[page, :, at % P] = v[b, t]
    if q is None:
        return None
    turned = q if frequencies is None else _turned(q, position, frequencies, interleaved)
    return torch.where(live[..., None, None], turned, torch.zeros_like(turned)).to(q.dtype)


# ---------------------------------------------------------------------------
# paged_attention_step
# ---------------------------------------------------------------------------


def paged_attention_step(q, k_cache, v_cache, pages, lengths, *, scale=None, window=None):
    """Attention of each sequence's newest token over its paged cache.

    ``o = sum_j w_j v_j`` with ``w`` the softmax of ``scale * (q . k_j)`` over the sequence's
    last ``window`` tokens (all without one), for each head; without gradients.  On the GPU the
    kernels take head sizes up to 256; larger ones run the eager body, with the warning of a
    decline.

    Parameters
    ----------
    q : (B, H, dk)
    k_cache : (N, Hk, P, dk)
    v_cache : (N, Hk, P, dv)
        ``Hk`` divides ``H``; each key head serves ``H / Hk`` heads in a row.  What lies in pages
        behind a sequence's last token, or before its window, has no part in the result,
        whatever it is; an infinity among the values that do have makes it infinite or NaN.  One
        type for ``q`` and the caches.
    pages : (B, M) integers
        Only the entries of tokens that are attended to are looked at.
    lengths : (B) integers
        Tokens of each sequence, the new one included.  Without any, ``o`` is 0.
    scale : float, optional
        ``dk ** -0.5`` by default.
    window : int, optional
        At least 1.

    Returns
    -------
    ``o`` (B, H, dv) in ``q``'s type.  A length beyond M pages, or a page that is not in the
    cache, raises ``IndexError`` in the eager body, on either device; with the kernels, where
    looking would wait for the GPU, that sequence's ``o`` is NaN.
    """
    what = "paged_attention_step"
    _check_one_type(what, q=q, k_cache=k_cache, v_cache=v_cache)
    _check_whole(what, q.device, pages=pages, lengths=lengths)
    qs = q.shape
    if len(qs) != 3:
        raise ValueError(f"{what}: q is (B, H, dk) (got {tuple(qs)})")
    B, H, dk = qs
    N, Hk, P, size, dv = _check_cache(what, k_cache, v_cache, pages, B)
    if size != dk or H < 1 or H % Hk:
        raise ValueError(f"{what}: q is {tuple(qs)}, the keys' heads {Hk} of size {size}; their "
                         "number divides q's, their size is q's")
    if lengths.shape != (B,):
        raise ValueError(f"{what}: lengths is (B,) = ({B},) (got {tuple(lengths.shape)})")
    if window is not None and (isinstance(window, bool) or int(window) != window or window < 1):
        raise ValueError(f"{what}: window is a whole number of at least 1 (got {window!r})")
    window = None if window is None else int(window)
    scale = dk**-0.5 if scale is None else float(scale)
    if B:
        out = _dispatch(what, q.is_cuda, lambda backend: backend.paged_attention_step_impl(
            q, k_cache, v_cache, pages, lengths, scale, window), "hip_decode")
        if out is not None:
            return out
    return _eager_attention(q, k_cache, v_cache, pages, lengths, scale, window)


@torch.no_grad()
def _eager_attention(q, k_cache, v_cache, pages, lengths, scale, window):
    what = "paged_attention_step"
    (B, H, dk), (N, Hk, P, dv) = q.shape, v_cache.shape
    if B == 0:
        return q.new_zeros(B, H, dv)
    lengths = lengths.long().clamp(min=0)
    n = int(lengths.max())
    if n > pages.shape[1] * P:
        raise IndexError(f"{what}: a sequence of {n} tokens is longer than its {pages.shape[1]} pages")
    if n == 0:
        return q.new_zeros(B, H, dv)
    at = torch.arange(n, device=q.device)
    live = at < lengths[:, None]
    if window is not None:
        live = live & (at >= lengths[:, None] - window)
    page = pages.long()[:, at // P]
    bad = live & ((page < 0) | (page >= N))
    if bool(bad.any()):
        raise IndexError(f"{what}: page {int(page[bad][0])} is outside of the cache of {N}")
    page = torch.where(live, page, torch.zeros_like(page))
    # (B, n, Hk, d), nothing of what is not attended to
    k, v = (torch.where(live[..., None, None], c[page, :, at % P], c.new_zeros(()))
            for c in (k_cache, v_cache))
    k, v = (_wide(c).transpose(1, 2) for c in (k, v))
    qw = _wide(q).view(B, Hk, H // Hk, dk) * scale
    with torch.autocast(q.device.type, enabled=False):  # it would round both products' operands
        scores = (qw @ k.transpose(-1, -2)).masked_fill(~live[:, None, None], -torch.inf)
        w = torch.softmax(scores, -1)
        w = w.masked_fill((lengths == 0)[:, None, None, None], 0)
        return (w @ v).reshape(B, H, dv).to(q.dtype)


# ---------------------------------------------------------------------------
# beam_select
# ---------------------------------------------------------------------------


def beam_select(logits, scores, width=None, *, end=None, finished=None):
    """A beam search's choice of the best continuations over beams and vocabulary.

    The candidate that goes on from beam ``k`` by token ``v`` has the score
    ``scores[b, k] + logits[b, k, v] - log(sum(exp(logits[b, k])))``, without gradients.

    Parameters
    ----------
    logits : (B, K, V)
        ``-inf`` for tokens that must not come.
    scores : (B, K)
        The beams' sums of log probabilities so far.
    width : int, optional
        Candidates to keep, K by default, at most K V.  On the GPU the kernels keep up to 64 of
        up to 256 beams; more run the eager body, with the warning of a decline.
    end : int, optional
        The token that ends a sequence.
    finished : (B, K) truth values, optional
        Beams that have ended, only with ``end``: such a beam has one candidate, ``end``, with
        the beam's own score; its logits are not read.

    Returns
    -------
    ``scores`` (B, width) in 32 bits (64 for float64 inputs), falling; ``parents`` and
    ``tokens`` (B, width) in int64; and, with ``end``, ``finished`` (B, width): whether the
    candidate's parent had ended or its token is ``end``.  Candidates are ranked by their scores
    in 64 bits, equal ones by the lower beam, then by the lower token.  On the GPU a beam's sum of
    exponentials is in 32 bits, some 2^-24 of it off and the same for beams of equal logits:
    candidates of other beams whose scores are that close may change places.  All candidates of a beam
    whose score or whose logits' sum is not finite (a NaN or ``inf`` among the logits, or only
    ``-inf``) have the score ``-inf``.
    """
    what = "beam_select"
    _check_floats(what, logits=logits, scores=scores)
    shape = logits.shape
    if len(shape) != 3 or scores.shape != shape[:2] or not (shape[1] and shape[2]):
        raise ValueError(f"{what}: logits is (B, K, V) and scores (B, K) (got "
                         f"{tuple(shape)} and {tuple(scores.shape)})")
    B, K, V = shape
    width = K if width is None else width
    if isinstance(width, bool) or int(width) != width or not 1 <= width <= K * V:
        raise ValueError(f"{what}: width is a whole number from 1 to K V = {K * V} (got {width!r})")
    width = int(width)
    if end is not None and (isinstance(end, bool) or int(end) != end or not 0 <= end < V):
        raise ValueError(f"{what}: end is a token from 0 to V - 1 = {V - 1} (got {end!r})")
    if finished is not None:
        if end is None:
            raise ValueError(f"{what}: finished beams go on by the token end, which is not given")
        if not torch.is_tensor(finished) or finished.dtype != torch.bool:
            raise TypeError(f"{what}: finished must be a tensor of truth values")
        if finished.shape != scores.shape or finished.device != logits.device:
            raise ValueError(f"{what}: finished is (B, K) on the logits' device (got "
                             f"{tuple(finished.shape)} on {finished.device})")
    if B:
        out = _dispatch(what, logits.is_cuda, lambda backend: backend.beam_select_impl(
            logits, scores, width, end, finished), "hip_decode")
        if out is not None:
            return out
    return _eager_select(logits, scores, width, end, finished)


@torch.no_grad()
def _eager_select(logits, scores, width, end, finished):
    V = logits.shape[2]
    wide = torch.promote_types(torch.promote_types(logits.dtype, scores.dtype), torch.float32)
    x, s = logits.double(), scores.double()
    if finished is not None:
        only = torch.full((V,), -torch.inf, dtype=x.dtype, device=x.device)
        only[int(end)] = 0.0
        x = torch.where(finished[..., None], only, x)
    x = x - x.amax(-1, keepdim=True)  # first of all: a large maximum would swallow the logarithm
    total = x.exp().sum(-1).log()
    dead = ~(torch.isfinite(total) & torch.isfinite(s))[..., None]
    score = (s[..., None] + (x - total[..., None])).masked_fill(dead, -torch.inf)
    score, order = torch.sort(score.flatten(1), dim=-1, descending=True, stable=True)
    order = order[:, :width]
    parent, token = order // V, order % V
    out = score[:, :width].to(wide), parent, token
    if end is None:
        return out
    done = token == int(end)
    return *out, done if finished is None else finished.gather(1, parent) | done


# ---------------------------------------------------------------------------
# reorder_states
# ---------------------------------------------------------------------------


def _leaves(states, out: list):
    """The tensors of nested lists, tuples and dicts, in order."""
    if torch.is_tensor(states):
        out.append(states)
    elif isinstance(states, (dict, list, tuple)):
        for s in states.values() if isinstance(states, dict) else states:
            if isinstance(s, torch.Tensor):
                out.append(s)
            else:
                _leaves(s, out)
    elif states is not None:
        raise TypeError("reorder_states: states are tensors, None, and lists, tuples and dicts of "
                        f"them (got {type(states).__name__})")
    return out


def _rebuilt(states, new):
    if torch.is_tensor(states):
        return next(new)
    if isinstance(states, dict):
        each = {k: _rebuilt(s, new) for k, s in states.items()}
        if type(states) is dict:
            return each
        out = copy.copy(states)  # a class of the caller's, with whatever else it holds
        for k, s in each.items():
            out[k] = s
        return out
    if isinstance(states, (list, tuple)):
        each = [next(new) if isinstance(s, torch.Tensor) else _rebuilt(s, new) for s in states]
        kind = type(states)
        if kind is list:
            return each
        if isinstance(states, list):
            out = copy.copy(states)
            out[:] = each
            return out
        return kind(*each) if hasattr(states, "_fields") else kind(each)
    return None


def reorder_states(states, parents):
    """Every state's rows in the order of the chosen beams, without gradients.

    Parameters
    ----------
    states : tensor, or nested lists, tuples and dicts of tensors and ``None``
        Each tensor is (B K, ...), of any type: row ``b K + k`` is beam ``k`` of search ``b``.
    parents : (B, W) integers
        ``W`` need not be ``K``: 0 for ``W`` beams out of each prompt.

    Returns
    -------
    The same structure, of the same classes, of new tensors (B W, ...): row ``b W + w`` is row ``b K + parents[b, w]``.
    A parent outside of 0 to K - 1 raises ``IndexError`` in the eager body, on either device; with
    the kernels, where looking would wait for the GPU, that row is 0.
    """
    what = "reorder_states"
    if not torch.is_tensor(parents):
        raise TypeError(f"{what}: parents must be a tensor of integers")
    _check_whole(what, parents.device, parents=parents)
    if parents.dim() != 2:
        raise ValueError(f"{what}: parents is (B, W) (got {tuple(parents.shape)})")
    B, W = parents.shape
    tensors = _leaves(states, [])
    if not tensors:
        return _rebuilt(states, iter(()))
    rows, device = tensors[0].shape[0] if tensors[0].dim() else -1, parents.device
    uneven = rows % B if B else rows
    for t in tensors:
        if t.device != device:
            raise ValueError(f"{what}: a state is on {t.device}, parents on {device}")
        shape = t.shape
        if uneven or not shape or shape[0] != rows:
            raise ValueError(f"{what}: each state has B K rows, the same for all, with B = {B} (got "
                             f"{tuple(t.shape)})")
    K = rows // B if B else 0
    if B * W:
        out = _dispatch(what, parents.is_cuda, lambda backend: backend.reorder_states_impl(
            tensors, parents, K), "hip_decode")
        if out is not None:
            return _rebuilt(states, iter(out))
    return _rebuilt(states, iter(_eager_reorder(tensors, parents, K)))


@torch.no_grad()
def _eager_reorder(tensors, parents, K):
    parents = parents.long()
    outside = (parents < 0) | (parents >= K)
    if bool(outside.any()):
        raise IndexError(f"reorder_states: parent {int(parents[outside][0])} is not one of {K} beams")
    rows = (parents + K * torch.arange(len(parents), device=parents.device)[:, None]).flatten()
    return [t[rows] for t in tensors]
