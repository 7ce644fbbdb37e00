"""Performance cases: the operators with which a language model answers.

Each case is a dict of plain values; ``op`` names the operator.

* ``append``: ``paged_cache_append``, new keys and values rotated by their positions and put
  into a paged cache, with the queries rotated on the way.
* ``attend``: ``paged_attention_step``, one new token of each sequence over a paged cache.
* ``beam``: ``beam_select``, a beam search's choice over beams and vocabulary.
* ``reorder``: ``reorder_states``, every layer's states follow the chosen beams.

The plain forms are elementary torch operations in 32 bits (angles and the sums that rank
candidates in 64).  ``exact`` evaluates the definitions in float64.
"""

from __future__ import annotations

import math

import torch

#: False: the plain forms.  True: the package's operators.
own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # The new token of every sequence of a serving batch: latency.
        dict(name="append-tokens", op="append", B=256, T=1, H=16, Hk=4, dk=128, dv=128, page=16,
             table=64, rotary=128, interleaved=False, dtype="bfloat16", ragged=False),
        # A batch of right-padded prompts behind what their pages already hold.
        dict(name="append-prompts", op="append", B=16, T=2048, H=16, Hk=8, dk=128, dv=128, page=64,
             table=40, rotary=128, interleaved=False, dtype="bfloat16", ragged=True),
        # Full precision, odd sizes, half of each head rotated, neighbours paired.
        dict(name="append-odd", op="append", B=5, T=333, H=6, Hk=3, dk=80, dv=48, page=7,
             table=61, rotary=40, interleaved=True, dtype="float32", ragged=True),
        # One sequence of a few thousand tokens: latency.
        dict(name="attend-single", op="attend", B=1, longest=4099, H=16, Hk=4, dk=128, dv=128,
             page=16, window=0, dtype="bfloat16", ragged=False),
        # A serving batch of sequences of many lengths, keys shared by groups of heads.
        dict(name="attend-batch", op="attend", B=64, longest=8192, H=16, Hk=4, dk=128, dv=128,
             page=16, window=0, dtype="bfloat16", ragged=True),
        # One very long sequence.
        dict(name="attend-long", op="attend", B=1, longest=524287, H=16, Hk=8, dk=128, dv=128,
             page=64, window=0, dtype="bfloat16", ragged=False),
        # Full precision, odd head sizes and pages, the last thousand tokens only.
        dict(name="attend-window-odd", op="attend", B=33, longest=5000, H=6, Hk=3, dk=80, dv=48,
             page=7, window=1000, dtype="float32", ragged=True),
        # Four beams of one sequence: latency.
        dict(name="beam-single", op="beam", B=1, K=4, width=4, V=50257, dtype="bfloat16",
             finished=0.0, masked=0.0),
        # A batch of searches, some beams at their end.
        dict(name="beam-batch", op="beam", B=64, K=8, width=8, V=50257, dtype="bfloat16",
             finished=0.2, masked=0.0),
        # Wide beams with as many candidates again, full precision, an odd vocabulary of which
        # half must not come next.
        dict(name="beam-wide", op="beam", B=16, K=16, width=32, V=32771, dtype="float32",
             finished=0.1, masked=0.5),
        # The matrix states of linear attention: 8 layers, 8 heads of 128 by 128.
        dict(name="reorder-matrices", op="reorder", B=16, K=8, width=8, layers=8, row=8 * 128 * 128,
             table=0, dtype="float32"),
        # The vector states of a recurrent stack and the sequences' page tables.
        dict(name="reorder-vectors", op="reorder", B=64, K=8, width=8, layers=24, row=1024,
             table=128, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("bfloat16", "bfloat16", "float16", "float32"))
    op = rng.choice(("append", "attend", "attend", "beam", "reorder"))
    if op == "append":
        Hk = rng.choice((1, 2, 3, 4, 8))
        T = rng.choice((1, 1, _log_int(rng, 2, 2048)))
        B = _log_int(rng, 1, min(256, max(1, 32768 // T)))
        dk = rng.choice((32, 64, 80, 96, 128, 192, 256))
        page = rng.choice((1, 7, 16, 32, 64))
        return dict(op=op, B=B, T=T, H=Hk * rng.choice((1, 2, 4)), Hk=Hk, dk=dk,
                    dv=rng.choice((dk, 64, 128)), page=page,
                    table=-(-(T + rng.randint(0, 1024)) // page),
                    rotary=rng.choice((dk, dk, dk // 2, 0)),
                    interleaved=rng.random() < 0.3, dtype=dtype,
                    ragged=T > 1 and rng.random() < 0.5)
    if op == "attend":
        Hk = rng.choice((1, 2, 3, 4, 8))
        dk = rng.choice((32, 64, 72, 80, 96, 128, 128, 192, 256))
        B = _log_int(rng, 1, 256)
        return dict(op=op, B=B, longest=_log_int(rng, 1, min(262144, 2**20 // B)),
                    H=Hk * rng.choice((1, 2, 4, 5, 8)), Hk=Hk, dk=dk,
                    dv=rng.choice((dk, dk, 64, 128)), page=rng.choice((1, 7, 16, 16, 64, 256)),
                    window=rng.choice((0, 0, _log_int(rng, 1, 4096))), dtype=dtype,
                    ragged=rng.random() < 0.7)
    if op == "beam":
        K = rng.choice((1, 2, 4, 5, 8, 16))
        V = _log_int(rng, 2000, 131072)
        return dict(op=op, B=_log_int(rng, 1, max(1, min(64, 2**25 // (K * V)))), K=K,
                    width=rng.choice((K, K, 2 * K, 4)), V=V, dtype=dtype,
                    finished=rng.choice((0.0, 0.3)), masked=rng.choice((0.0, 0.5)))
    layers = _log_int(rng, 1, 48)
    K, B = rng.choice((1, 2, 4, 8)), _log_int(rng, 1, 64)
    most = 2**27 // (layers * B * K)
    return dict(op=op, B=B, K=K, width=rng.choice((K, K, 2 * K)), layers=layers,
                row=_log_int(rng, 1, most), table=rng.choice((0, _log_int(rng, 1, 512))),
                dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(self, *shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=self.g) * std).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)

    def integers(self, low, high, *shape):
        return torch.randint(low, high, shape, device="cuda", generator=self.g)

    def tables(self, B, M, used):
        """Page tables (B, M) over B M pages in no order; entries past a sequence's ``used``
        tables are -1."""
        at = torch.randperm(B * M, device="cuda", generator=self.g).view(B, M).to(torch.int32)
        return torch.where(torch.arange(M, device="cuda") < used[:, None], at, at.new_tensor(-1))


def _prepare_append(case, r):
    dtype = DTYPES[case["dtype"]]
    B, T, H, Hk, dk, dv, P, M = (case[n] for n in ("B", "T", "H", "Hk", "dk", "dv", "page", "table"))
    room = M * P - T
    s = dict(
        q=r.normal(B, T, H, dk, dtype=dtype),
        k=r.normal(B, T, Hk, dk, dtype=dtype),
        v=r.normal(B, T, Hk, dv, dtype=dtype),
        k_cache=r.normal(B * M, Hk, P, dk, dtype=dtype),
        v_cache=r.normal(B * M, Hk, P, dv, dtype=dtype),
        start=r.integers(0, room + 1, B).to(torch.int32),
        lengths=None,
        frequencies=None,
    )
    if case["ragged"]:
        s["lengths"] = r.integers(0, T + 1, B).to(torch.int32)
        s["lengths"][0] = T
    if case["rotary"]:
        n = case["rotary"]
        s["frequencies"] = 10000.0 ** (-torch.arange(0, n, 2, device="cuda").float() / n)
    count = T if s["lengths"] is None else s["lengths"]
    s["pages"] = r.tables(B, M, (s["start"] + count + P - 1) // P)
    return s


def _prepare_attend(case, r):
    dtype = DTYPES[case["dtype"]]
    B, n, H, Hk, dk, dv, P = (case[x] for x in ("B", "longest", "H", "Hk", "dk", "dv", "page"))
    lengths = torch.full((B,), n, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        lengths = r.integers(0, n + 1, B).to(torch.int32)
        lengths[-1] = n
    M = -(-n // P)
    return dict(
        q=r.normal(B, H, dk, dtype=dtype, std=1.5),
        k_cache=r.normal(B * M, Hk, P, dk, dtype=dtype),
        v_cache=r.normal(B * M, Hk, P, dv, dtype=dtype),
        pages=r.tables(B, M, (lengths + P - 1) // P),
        lengths=lengths,
    )


def _prepare_beam(case, r):
    B, K, V = case["B"], case["K"], case["V"]
    logits = r.normal(B, K, V, dtype=DTYPES[case["dtype"]], std=2.5)
    if case["masked"]:
        logits.masked_fill_(r.uniform(B, 1, V) < case["masked"], -math.inf)
    return dict(
        logits=logits,
        scores=-5.0 - 10.0 * r.uniform(B, K),
        finished=r.uniform(B, K) < case["finished"] if case["finished"] else None,
    )


def _prepare_reorder(case, r):
    rows = case["B"] * case["K"]
    states = [r.normal(rows, case["row"], dtype=DTYPES[case["dtype"]])
              for _ in range(case["layers"])]
    if case["table"]:
        states.append(r.integers(0, 1 << 20, rows, case["table"]).to(torch.int32))
    return dict(states=states, parents=r.integers(0, case["K"], case["B"], case["width"]))


_PREPARE = {"append": _prepare_append, "attend": _prepare_attend, "beam": _prepare_beam,
            "reorder": _prepare_reorder}


def prepare(case, seed):
    return dict(_PREPARE[case["op"]](case, _Rand(seed)), case=case)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _rotated(x, position, frequencies, interleaved):
    """x (B, T, heads, d) turned by its positions (B, T), in 32 bits."""
    x = x.float()
    if frequencies is None:
        return x
    n = 2 * frequencies.numel()
    angle = position.double()[..., None] * frequencies.double()
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    part, rest = x[..., :n], x[..., n:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., : n // 2], part[..., n // 2 :]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _plain_append(case, s):
    B, T = s["k"].shape[:2]
    P, dtype = case["page"], s["k"].dtype
    t = torch.arange(T, device="cuda").expand(B, T)
    position = s["start"][:, None] + t
    q = _rotated(s["q"], position, s["frequencies"], case["interleaved"])
    k = _rotated(s["k"], position, s["frequencies"], case["interleaved"]).to(dtype)
    v = s["v"]
    if s["lengths"] is None:
        page, slot = s["pages"].gather(1, (position // P).long()).flatten(), (position % P).flatten()
        k, v = k.flatten(0, 1), v.flatten(0, 1)
    else:
        live = t < s["lengths"][:, None]
        q = torch.where(live[..., None, None], q, torch.zeros_like(q))
        b, t = torch.nonzero(live, as_tuple=True)
        position = position[b, t].long()
        page, slot = s["pages"][b, position // P], position % P
        k, v = k[b, t], v[b, t]
    s["k_cache"][page.long(), :, slot.long()] = k
    s["v_cache"][page.long(), :, slot.long()] = v
    return q.to(dtype), s["k_cache"], s["v_cache"]


def _plain_attend(case, s):
    q, pages, lengths = s["q"], s["pages"], s["lengths"]
    B, H, dk = q.shape
    N, Hk, P, dv = s["v_cache"].shape
    n = pages.shape[1] * P

    def rows(cache):
        cache = cache[pages.clamp(min=0).long()].float()
        return cache.transpose(1, 2).reshape(B, Hk, n, -1)

    at = torch.arange(n, device="cuda")
    live = at < lengths[:, None]
    if case["window"]:
        live = live & (at >= lengths[:, None] - case["window"])
    live = live[:, None, None, :]
    scores = (q.float().view(B, Hk, H // Hk, dk) * dk**-0.5) @ rows(s["k_cache"]).transpose(-1, -2)
    scores = torch.where(live, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total == 0, torch.ones_like(total), total)
    return (e @ rows(s["v_cache"])).view(B, H, dv).to(q.dtype)


_END = 2


def _plain_beam(case, s):
    B, K, V = s["logits"].shape
    W = case["width"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    total = torch.exp(x - top).sum(-1, keepdim=True, dtype=torch.float64)
    norm = top.double() + torch.log(total)
    if s["finished"] is not None:  # such a beam goes on by its end alone, at no cost
        done = s["finished"][..., None]
        only = torch.where(torch.arange(V, device="cuda") == _END, 0.0, -math.inf)
        x = torch.where(done, only, x)
        norm = torch.where(done, torch.zeros_like(norm), norm)
    # A row's candidates by their logits, equal ones by their tokens: whole numbers in that order.
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * 2**32 + (
        2**32 - 1 - torch.arange(V, device="cuda"))
    token = (2**32 - 1 - (torch.topk(key, min(W, V), -1).values & 0xFFFFFFFF)).flatten(1)
    n = min(W, V)
    parent = torch.arange(K, device="cuda").repeat_interleave(n).expand(B, K * n)
    score = s["scores"].double()[..., None] + (x.gather(-1, token.view(B, K, n)).double() - norm)
    score, order = torch.sort(score.flatten(1), dim=-1, descending=True, stable=True)
    order = order[:, :W]
    parent, token = parent.gather(1, order), token.gather(1, order)
    out = score[:, :W].float(), parent, token
    if s["finished"] is None:
        return out
    return *out, s["finished"].gather(1, parent) | (token == _END)


def _plain_reorder(case, s):
    parents = s["parents"]
    rows = (parents + case["K"] * torch.arange(case["B"], device="cuda")[:, None]).flatten()
    return [t.index_select(0, rows) for t in s["states"]]


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "beam": _plain_beam,
          "reorder": _plain_reorder}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


@torch.no_grad()
def run(s):
    case = s["case"]
    if not own:
        return _PLAIN[case["op"]](case, s)
    import mingru_amd

    if case["op"] == "append":
        q = mingru_amd.paged_cache_append(
            s["k"], s["v"], s["k_cache"], s["v_cache"], s["pages"], s["start"], q=s["q"],
            lengths=s["lengths"], frequencies=s["frequencies"], interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if case["op"] == "attend":
        return mingru_amd.paged_attention_step(s["q"], s["k_cache"], s["v_cache"], s["pages"],
                                               s["lengths"], window=case["window"] or None)
    if case["op"] == "beam":
        return mingru_amd.beam_select(s["logits"], s["scores"], case["width"],
                                      end=None if s["finished"] is None else _END,
                                      finished=s["finished"])
    return mingru_amd.reorder_states(s["states"], s["parents"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "append":
        tokens = case["B"] * case["T"]
        one = (case["H"] + case["Hk"]) * case["dk"] + case["Hk"] * case["dv"]
        # Half of a ragged batch's tokens are there.
        share = 0.5 + 0.5 / case["B"] if case["ragged"] else 1.0
        return {"bytes": 2 * e * tokens * one * share,
                "flops": 3.0 * tokens * share * (case["H"] + case["Hk"]) * case["rotary"]}
    if case["op"] == "attend":
        n, B = case["longest"], case["B"]
        live = n if not case["window"] else min(n, case["window"])
        tokens = B * live
        if case["ragged"]:  # lengths from 0 to the longest, one of them the longest
            tokens = live + (B - 1) * (live - live * live / (2.0 * n))
        heads = case["Hk"] * (case["dk"] + case["dv"])
        return {"bytes": e * (tokens * heads + B * case["H"] * (case["dk"] + case["dv"])),
                "flops": 2.0 * tokens * case["H"] * (case["dk"] + case["dv"])}
    if case["op"] == "beam":
        B, K, V, W = case["B"], case["K"], case["V"], case["width"]
        read = B * K * V * (1.0 - case["finished"])
        return {"bytes": read * e + 5 * B * K + 21 * B * W, "flops": 4.0 * read}
    rows = case["B"] * case["width"]
    return {"bytes": 2 * rows * (case["layers"] * case["row"] * e + 4 * case["table"]) + 8 * rows,
            "flops": 0.0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_append(case, s):
    P = case["page"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    B, T = k.shape[:2]
    start = s["start"].tolist()
    counts = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = counts[b]
        at = start[b] + torch.arange(T, device="cuda")
        if s["frequencies"] is not None:
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               at.double()[:, None] * s["frequencies"].double())[:, None]
            r = case["rotary"]
            for x in (q, k):
                if case["interleaved"]:
                    z = torch.complex(x[b, ..., 0:r:2], x[b, ..., 1:r:2]) * turn
                    x[b, ..., 0:r:2], x[b, ..., 1:r:2] = z.real, z.imag
                else:
                    z = torch.complex(x[b, ..., : r // 2], x[b, ..., r // 2 : r]) * turn
                    x[b, ..., : r // 2], x[b, ..., r // 2 : r] = z.real, z.imag
        q[b, n:] = 0
        page, slot = s["pages"][b][at[:n] // P].long(), at[:n] % P
        kc[page, :, slot], vc[page, :, slot] = k[b, :n], v[b, :n]
    return q, kc, vc


def _exact_attend(case, s):
    q, dk = s["q"].double(), case["dk"]
    B, H = q.shape[:2]
    P, Hk = case["page"], case["Hk"]
    out = torch.zeros(B, H, case["dv"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == first:
            continue
        at = torch.arange(first, n, device="cuda")
        page, slot = s["pages"][b][at // P].long(), at % P
        for h in range(Hk):
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            k, v = (s[c][page, h, slot].double() for c in ("k_cache", "v_cache"))
            out[b, heads] = torch.softmax(q[b, heads] @ k.t() / math.sqrt(dk), -1) @ v
    return out


def _exact_beam(case, s):
    B, K, V = s["logits"].shape
    W = case["width"]
    parts = []
    for b in range(B):
        x = torch.log_softmax(s["logits"][b].double(), -1)
        if s["finished"] is not None:
            done = s["finished"][b]
            x[done] = -math.inf
            x[done, _END] = 0.0
        every = (s["scores"][b].double()[:, None] + x).flatten()
        least = torch.topk(every, W).values[-1]
        at = torch.nonzero(every >= least)[:, 0]  # in the order of beams and tokens
        order = torch.sort(every[at], dim=-1, descending=True, stable=True).indices[:W]
        parts.append((every[at][order], at[order] // V, at[order] % V))
    score, parent, token = (torch.stack(p) for p in zip(*parts))
    if s["finished"] is None:
        return score, parent, token
    return score, parent, token, s["finished"].gather(1, parent) | (token == _END)


def _exact_reorder(case, s):
    B, K, W = case["B"], case["K"], case["width"]
    out = []
    for t in s["states"]:
        t = t.view(B, K, -1)
        t = torch.stack([t[b, s["parents"][b]] for b in range(B)]).view(B * W, -1)
        out.append(t.double() if t.dtype.is_floating_point else t)
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    return _exact_beam(case, s) if case["op"] == "beam" else _exact_reorder(case, s)
