"""The operators that serve many requests from a paged KV cache of 16 bits: appending keys and values
to their pages with the rotation on the way, attention over the pages (single tokens, a few, whole
chunks of prompts), attention of a batch whose requests share a long prefix, and attention over the
pages that a cheap score selects.

Every case is one pass as a serving program makes it for one layer: ``run`` calls
``HipDecodeBackend`` where ``own`` is true and computes the same formulas with elementary torch
operations where it is false.  ``exact`` restates them in float64.

The cache: ``k_pages`` and ``v_pages`` [pages, kv_heads, page, head_dim]; token t of row r lies in page
``table[r, t // page]``, slot ``t % page``.  ``k_bounds`` [pages, kv_heads, 2, head_dim] holds, for every
dim, the least and the greatest value among a page's keys.
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_MAX_APPEND = 16384 * (64 + 2 * 8) * 128          # values of the largest append
_MAX_CACHE = 8 * 65536 * 10 * 128                 # K values of the largest cache
_MAX_PRODUCTS = 8 * 10 ** 8 * 128                 # (query head, visible token) pairs x head_dim


def listed() -> list[dict]:
    return [
        # one new token for each of eight requests of a 1B model: the smallest append of a decode step
        {"name": "append-step", "kind": "append", "rows": 8, "tokens": 1, "ragged": False, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "page": 16, "rotary": 64, "interleaved": False, "start": 575, "bounds": False, "dtype": "f16"},
        # a step that mixes decoding requests, chunks of prompts and idle rows; half of a head turned, page bounds kept
        {"name": "append-mixed", "kind": "append", "rows": 12, "tokens": 517, "ragged": True, "heads": 40, "kv_heads": 10,
         "head_dim": 128, "page": 64, "rotary": 64, "interleaved": True, "start": 4001, "bounds": True, "dtype": "bf16"},
        # one long prompt that begins inside a page
        {"name": "append-prompt", "kind": "append", "rows": 1, "tokens": 16384, "ragged": False, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "page": 128, "rotary": 128, "interleaved": False, "start": 5, "bounds": True, "dtype": "f16"},
        # one token of one request, a few hundred tokens behind it: latency
        {"name": "paged-step", "kind": "paged", "rows": 1, "length": 575, "tokens": 1, "ragged": False, "heads": 32,
         "kv_heads": 8, "head_dim": 64, "page": 16, "window": 0, "sinks": False, "dtype": "f16"},
        # 32 requests of unequal length, one token each, an idle row among them: the cache read once
        {"name": "paged-batch", "kind": "paged", "rows": 32, "length": 8001, "tokens": 1, "ragged": True, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0, "sinks": False, "dtype": "bf16"},
        # four drafted tokens of each of sixteen requests, to be verified
        {"name": "paged-draft", "kind": "paged", "rows": 16, "length": 4001, "tokens": 4, "ragged": False, "heads": 40,
         "kv_heads": 10, "head_dim": 128, "page": 16, "window": 0, "sinks": False, "dtype": "f16"},
        # chunks of four prompts in a layer with a window of 128 tokens and sinks
        {"name": "paged-window", "kind": "paged", "rows": 4, "length": 4099, "tokens": 1027, "ragged": True, "heads": 64,
         "kv_heads": 8, "head_dim": 64, "page": 32, "window": 128, "sinks": True, "dtype": "f16"},
        # chunks of up to 2048 tokens of prompts that already hold thousands: the most products
        {"name": "paged-chunk", "kind": "paged", "rows": 4, "length": 8192, "tokens": 2048, "ragged": True, "heads": 40,
         "kv_heads": 10, "head_dim": 128, "page": 64, "window": 0, "sinks": False, "dtype": "bf16"},
        # eight requests of a 1B model behind one prompt of two thousand tokens
        {"name": "shared-few", "kind": "paged", "rows": 8, "length": 2309, "tokens": 1, "ragged": True, "heads": 32,
         "kv_heads": 8, "head_dim": 64, "page": 16, "window": 0, "sinks": False, "shared": 2048, "dtype": "f16"},
        # 64 requests behind one document of 32768 tokens
        {"name": "shared-batch", "kind": "paged", "rows": 64, "length": 33601, "tokens": 1, "ragged": True, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0, "sinks": False, "shared": 32768, "dtype": "bf16"},
        # one request at 32000 tokens that reads 64 of its 500 pages
        {"name": "sparse-step", "kind": "sparse", "rows": 1, "length": 32000, "ragged": False, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "page": 64, "count": 64, "first": 1, "last": 2, "dtype": "f16"},
        # eight requests of up to 65536 tokens, each reading a sixteenth of its pages
        {"name": "sparse-batch", "kind": "sparse", "rows": 8, "length": 65536, "ragged": True, "heads": 40, "kv_heads": 10,
         "head_dim": 128, "page": 32, "count": 128, "first": 2, "last": 4, "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "paged", "paged", "shared", "sparse"])
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "ragged": rng.random() < 0.6, "dtype": rng.choice(["f16", "bf16"])}
    if kind == "append":
        rows = _log_int(rng, 1, 64)
        most = max(1, min(16384, _MAX_APPEND // (rows * (heads + 2 * kv_heads) * head_dim)))
        return {**case, "rows": rows, "tokens": _log_int(rng, 1, most), "start": rng.randint(0, 9000),
                "rotary": rng.choice([head_dim // 4, head_dim // 2, head_dim]), "interleaved": rng.random() < 0.4,
                "bounds": rng.random() < 0.5}
    rows = _log_int(rng, 1, 64)
    most = min(65536, _MAX_CACHE // (rows * kv_heads * head_dim))
    length = _log_int(rng, 1, most)
    if kind == "sparse":
        first, last = rng.choice([0, 1, 2]), rng.choice([0, 1, 4])
        return {**case, "rows": rows, "length": length, "count": first + last + _log_int(rng, 1, 128), "first": first, "last": last}
    tokens = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 1, 2048)])
    tokens = max(1, min(tokens, length, _MAX_PRODUCTS // (rows * length * heads * head_dim)))
    if kind == "shared":
        length = _log_int(rng, 2 * page, max(2 * page, min(33601, most)))
        tokens = 1 if rng.random() < 0.7 else min(tokens, 4)
        while rows * tokens * length * heads * head_dim > _MAX_PRODUCTS:
            rows = max(1, rows // 2)
            if rows == 1:
                tokens = 1
        return {**case, "kind": "paged", "rows": rows, "length": length, "tokens": tokens, "window": 0,
                "sinks": rng.random() < 0.3, "shared": rng.randint(1, length // page) * page}
    return {**case, "rows": rows, "length": length, "tokens": tokens,
            "window": rng.choice([0, 0, _log_int(rng, 16, 4096)]), "sinks": rng.random() < 0.4}


# ------------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype).mul_(std)


def _counts(case: dict) -> list[int]:
    """New (or query) tokens of every row: the case's own first, then chunks, single tokens and none."""
    n, rows = case.get("tokens", 1), case["rows"]
    if not case["ragged"] or n == 1:
        return [n] * rows
    return [n if r == 0 else 1 if r % 4 == 2 else 0 if r % 8 == 5 else max(1, n * ((7 * r) % rows) // rows) for r in range(rows)]


def _lengths(case: dict) -> list[int]:
    """Tokens that a row holds, its new ones included: the case's own first, down to about a third of it
    (behind a shared prefix, a third of what follows that), an idle row in larger batches."""
    n, rows, base = case["length"], case["rows"], case.get("shared", 0)
    if not case["ragged"]:
        return [n] * rows
    own_part = n - base
    return [0 if r % 16 == 11 else max(1, base + own_part - 2 * own_part * r // (3 * rows)) for r in range(rows)]


def _shared_pages(case: dict) -> int:
    return case.get("shared", 0) // case["page"]


def _visible(case: dict) -> list[tuple[int, int, int]]:
    """(row, first, past the last visible token) of every query."""
    out = []
    for r, (n, t) in enumerate(zip(_lengths(case), _counts(case))):
        for i in range(t):
            hi = max(0, n - (t - 1 - i))
            out.append((r, max(0, hi - case["window"]) if case.get("window") else 0, hi))
    return out


def _table(g, needs: list[int], shared: int, pages: int):
    """A table of distinct, scattered pages; the first `shared` are the same for every row.  Entries that
    no token needs are 0."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(needs), max(max(needs), shared, 1)), device="cuda", dtype=torch.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for r, n in enumerate(needs):
        own_pages = max(0, n - shared)
        table[r, shared:shared + own_pages] = order[at:at + own_pages]
        at += own_pages
    return table


def prepare(case: dict, seed: int) -> dict:
    g, kind, dt = _gen(seed), case["kind"], _DTYPES[case["dtype"]]
    h, kvh, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    counts = _counts(case)
    starts = [max(0, case["start"] - 37 * r) for r in range(case["rows"])] if kind == "append" else []
    held = [s + n for s, n in zip(starts, counts)] if kind == "append" else _lengths(case)
    needs, shared = [-(-n // page) for n in held], _shared_pages(case)
    pages = shared + sum(max(0, n - shared) for n in needs) + 3
    state = {"case": case, "table": _table(g, needs, shared, pages)}
    # keys with a spread of channel means, values without, as attention layers make them
    means = _normal(g, (1, kvh, 1, d), std=1.5)
    state["k_pages"] = _normal(g, (pages, kvh, page, d), dt).add_(means.to(dt))
    state["v_pages"] = _normal(g, (pages, kvh, page, d), dt)
    if kind == "sparse" or case.get("bounds"):
        state["k_bounds"] = torch.stack((state["k_pages"].amin(2), state["k_pages"].amax(2)), 2)
    total = sum(counts)
    if case["ragged"] and case.get("tokens", 1) > 1:           # (as many tokens for every row otherwise)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        state["cu"] = torch.tensor(cu, device="cuda", dtype=torch.int32)
    if kind == "append":
        # parts of one projection's output, as a fused QKV product leaves them
        qkv = _normal(g, (total, (h + 2 * kvh) * d)).view(total, h + 2 * kvh, d)
        qkv[:, h:h + kvh] += means[:, :, 0]
        qkv = qkv.to(dt)
        state["q"], state["k"], state["v"] = qkv[:, :h], qkv[:, h:h + kvh], qkv[:, h + kvh:]
        state["starts"] = torch.tensor(starts, device="cuda", dtype=torch.int32)
        r = case["rotary"]
        state["inv_freq"] = 500000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        state["q_out"] = torch.empty((total, h, d), device="cuda", dtype=dt)
        return state
    state["q"] = _normal(g, (total, h, d), dt)
    state["lengths"] = torch.tensor(held, device="cuda", dtype=torch.int32)
    state["out"] = torch.empty_like(state["q"])
    state["sinks"] = _normal(g, (h,), dt) if case.get("sinks") else None
    if kind == "sparse":
        state["selected"] = torch.empty((case["rows"], kvh, case["count"]), device="cuda", dtype=torch.int32)
    return state


# ------------------------------------------------------------------------------- the framework's calls
@functools.lru_cache(maxsize=None)
def _backend():
    from thintensor_amd.backend import HipDecodeBackend

    return HipDecodeBackend(torch.device("cuda:0"), torch.float16, 2048, 2048, 512, 8192)


def _own_cache(state):
    if "handle" not in state:                 # the object that a program makes once around a cache's tensors
        from thintensor_amd.paged_cache import PagedKvCache

        state["handle"] = PagedKvCache(state["k_pages"], state["v_pages"], state.get("k_bounds"))
    return state["handle"]


def _run_own(state):
    case, be, cache = state["case"], _backend(), _own_cache(state)
    if case["kind"] == "append":
        be.rotary_append_paged(cache, state["q"], state["k"], state["v"], state["table"], state["starts"],
                               state["inv_freq"], state["q_out"], cu_tokens=state.get("cu"),
                               interleaved=case["interleaved"])
        held = (state["q_out"], state["k_pages"], state["v_pages"])
        return (*held, state["k_bounds"]) if case["bounds"] else held
    if case["kind"] == "sparse":
        be.select_pages(state["q"], cache, state["table"], state["lengths"], state["selected"],
                        first_pages=case["first"], last_pages=case["last"])
        be.gqa_attention_paged(state["q"], cache, state["table"], state["lengths"], state["out"],
                               selected=state["selected"])
        return state["selected"], state["out"]
    return be.gqa_attention_paged(state["q"], cache, state["table"], state["lengths"], state["out"],
                                  cu_tokens=state.get("cu"), shared_pages=_shared_pages(case),
                                  window=case["window"], sinks=state["sinks"])


# ------------------------------------------------------------------------------- the plain forms
def _token_rows(state):
    """Row and place in it of every token."""
    total, rows = state["q"].shape[0], state["case"]["rows"]
    t = torch.arange(total, device="cuda")
    if "cu" not in state:
        return t // (total // rows), t % (total // rows)
    cu = state["cu"].long()
    row = (t[:, None] >= cu[None, 1:]).sum(1)
    return row, t - cu[row]


def _rotate(x, cos, sin, rotary, interleaved):
    head, rest = x[..., :rotary].float(), x[..., rotary:].float()
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : rotary // 2], head[..., rotary // 2:])
    c, s = cos[:, None], sin[:, None]
    first, second = a * c - b * s, b * c + a * s
    head = torch.stack((first, second), -1).flatten(-2) if interleaved else torch.cat((first, second), -1)
    return torch.cat((head, rest), -1).to(x.dtype)


def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    row, i = _token_rows(state)
    pos = state["starts"].long()[row] + i
    angle = pos.double()[:, None] * state["inv_freq"]          # far positions: angles in 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotate(state["q"], cos, sin, case["rotary"], case["interleaved"])
    k = _rotate(state["k"], cos, sin, case["rotary"], case["interleaved"])
    at, slot = state["table"].long()[row, pos // page], pos % page
    state["k_pages"][at, :, slot] = k
    state["v_pages"][at, :, slot] = state["v"]
    if not case["bounds"]:
        return q, state["k_pages"], state["v_pages"]
    bounds = state["k_bounds"].float()
    index = at[:, None, None].expand(k.shape)
    for side, extreme, empty in ((0, "amin", math.inf), (1, "amax", -math.inf)):
        part = bounds[:, :, side].contiguous()
        part[at[slot == 0]] = empty                            # a page that begins anew
        bounds[:, :, side] = part.scatter_reduce_(0, index, k.float(), extreme)
    state["k_bounds"].copy_(bounds)
    return q, state["k_pages"], state["v_pages"], state["k_bounds"]


def _attend(q, k, v, seen, sinks):
    """q [KVH, M, D], k and v [KVH, N, D] in 32 bits, seen [M, N] (or [KVH, 1, N]), sinks [KVH, M] or None."""
    s = torch.matmul(q, k.transpose(1, 2).contiguous()) * q.shape[-1] ** -0.5
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(2, keepdim=True)
    if sinks is not None:
        top = torch.maximum(top, sinks[..., None])
    top = torch.where(top == -math.inf, 0.0, top)              # a query that sees nothing
    p = torch.exp(s - top)
    total = p.sum(2, keepdim=True)
    nothing = total == 0 if sinks is None else (s == -math.inf).all(2, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks[..., None] - top)
    return torch.where(nothing, 0.0, torch.matmul(p, v) / torch.where(nothing, 1.0, total))


def _plain_attention(state, pages_of=None):
    case, q = state["case"], state["q"]
    kvh, d, page, h = case["kv_heads"], case["head_dim"], case["page"], case["heads"]
    g = h // kvh
    out = torch.zeros(q.shape, device="cuda")
    at = 0
    for r, (n, t) in enumerate(zip(_lengths(case), _counts(case))):
        if t == 0 or n == 0:
            at += t
            continue
        qr = q[at:at + t].float().view(t, kvh, g, d).permute(1, 0, 2, 3)                     # [KVH, t, g, D]
        place = torch.arange(t, device="cuda").repeat_interleave(g)
        hi = n - (t - 1 - place)
        lo = (hi - case["window"]).clamp_min(0) if case.get("window") else torch.zeros_like(hi)
        sinks = state["sinks"] if case["kind"] == "paged" else None
        if sinks is not None:
            sinks = sinks.float().view(kvh, 1, g).expand(kvh, t, g).reshape(kvh, t * g)
        if pages_of is not None:
            logical = pages_of[r].long()                                                     # [KVH, count], -1: none
            ids = state["table"][r].long()[logical.clamp_min(0)]
            heads = torch.arange(kvh, device="cuda")[:, None]
            k, v = (state[name][ids, heads].flatten(1, 2).float() for name in ("k_pages", "v_pages"))
            token = (logical[..., None] * page + torch.arange(page, device="cuda")).flatten(1)
            seen = (token < n) & (logical >= 0).repeat_interleave(page, 1)
            out[at:at + t] = _attend(qr.reshape(kvh, t * g, d), k, v, seen[:, None], sinks).view(t, h, d)
        else:
            first = max(0, n - t + 1 - case["window"]) // page if case["window"] else 0
            ids = state["table"][r, first:-(-n // page)].long()
            token = torch.arange(first * page, first * page + len(ids) * page, device="cuda")
            seen = (token >= lo[:, None]) & (token < hi[:, None])
            # one KV head at a time where the scores of all would take much memory
            step = 1 if t * h * len(token) > 1 << 28 else kvh
            for j in range(0, kvh, step):
                k, v = (state[name][:, j:j + step][ids].transpose(0, 1).flatten(1, 2).float() for name in ("k_pages", "v_pages"))
                o = _attend(qr[j:j + step].reshape(step, t * g, d), k, v, seen, None if sinks is None else sinks[j:j + step])
                out[at:at + t].view(t, kvh, g, d)[:, j:j + step] = o.view(step, t, g, d).transpose(0, 1)
        at += t
    return out.to(q.dtype)


def _plain_select(state):
    """Scores in 64 bits (one decides which page is read), rounded to 32 as the operator's are."""
    case, page = state["case"], state["case"]["page"]
    kvh, d, count = case["kv_heads"], case["head_dim"], case["count"]
    selected = torch.full_like(state["selected"], -1)
    for r, n in enumerate(_lengths(case)):
        pages = -(-n // page)
        if pages == 0:
            continue
        q = state["q"][r].double().view(kvh, -1, d)
        b = state["k_bounds"][state["table"][r, :pages].long()].double().permute(1, 2, 0, 3)  # [KVH, 2, pages, D]
        s = torch.stack([torch.maximum(b[:, 0] * q[:, j, None], b[:, 1] * q[:, j, None]).sum(-1)
                         for j in range(q.shape[1])]).amax(0).float()
        s[:, :case["first"]] = math.inf
        s[:, max(0, pages - case["last"]):] = math.inf
        order = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :count]         # ties: the lowest page
        selected[r, :, :order.shape[1]] = torch.sort(order, dim=1).values.to(torch.int32)
    return selected


def run(state: dict):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _plain_append(state)
    if kind == "sparse":
        selected = _plain_select(state)
        return selected, _plain_attention(state, selected)
    return _plain_attention(state)


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    h, kvh, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    counts = _counts(case)
    total = sum(counts)
    if case["kind"] == "append":
        held = [max(0, case["start"] - 37 * r) for r in range(case["rows"])]
        touched = sum((s + n - 1) // page - s // page + 1 for s, n in zip(held, counts) if n)
        bounds = 2 * touched * kvh * 2 * d * 2 if case["bounds"] else 0
        return {"bytes": 2 * total * (h + 2 * kvh) * d * 2 + bounds, "flops": 3 * total * (h + kvh) * case["rotary"]}
    io = 2 * total * h * d * 2
    if case["kind"] == "sparse":
        pages = [-(-n // page) for n in _lengths(case)]
        read = [min(n, min(p, case["count"]) * page) for n, p in zip(_lengths(case), pages)]
        return {"bytes": sum(pages) * kvh * 2 * d * 2 + sum(read) * kvh * d * 4 + io,
                "flops": 3 * sum(pages) * h * d + 4 * sum(read) * h * d}
    shared, reach, pairs = _shared_pages(case) * page, {}, 0
    for r, lo, hi in _visible(case):
        pairs += hi - lo
        if hi > lo:
            a, b = reach.get(r, (lo, hi))
            reach[r] = (min(a, lo), max(b, hi))
    tokens = sum(max(0, b - max(a, shared)) for a, b in reach.values())
    inside = [(min(a, shared), min(b, shared)) for a, b in reach.values()]
    if inside:
        tokens += max(b for _, b in inside) - min(a for a, _ in inside)
    return {"bytes": tokens * kvh * d * 4 + io, "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------------------- float64, from the definitions
def _exact_append(state):
    case, page = state["case"], state["case"]["page"]
    counts, table = _counts(case), state["table"].cpu().numpy()
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    bounds = state["k_bounds"].double() if case["bounds"] else None
    r = case["rotary"]
    pairs = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    qs, at = [], 0
    for row, n in enumerate(counts):
        start = int(state["starts"][row])
        turn = torch.arange(start, start + n, device="cuda").double()[:, None] * state["inv_freq"]
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]
        turned = []
        for x in (state["q"], state["k"]):
            x = x[at:at + n].double()
            z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * turn
            x = x.clone()
            x[..., pairs[0]], x[..., pairs[1]] = z.real, z.imag
            turned.append(x)
        qs.append(turned[0])
        t = 0
        while t < n:                                           # one run of tokens inside a page after another
            slot = (start + t) % page
            m = min(n - t, page - slot)
            p = int(table[row, (start + t) // page])
            keys = turned[1][t:t + m]
            k_pages[p, :, slot:slot + m] = keys.transpose(0, 1)
            v_pages[p, :, slot:slot + m] = state["v"][at + t:at + t + m].double().transpose(0, 1)
            if bounds is not None:
                lo, hi = keys.min(0).values, keys.max(0).values
                bounds[p, :, 0] = torch.minimum(bounds[p, :, 0], lo) if slot else lo
                bounds[p, :, 1] = torch.maximum(bounds[p, :, 1], hi) if slot else hi
            t += m
        at += n
    out = (torch.cat(qs), k_pages, v_pages)
    return out if bounds is None else (*out, bounds)


def _exact_attention(state, pages_of=None):
    """One query head at a time over the tokens it sees, gathered by number."""
    case, page = state["case"], state["case"]["page"]
    kvh, d, window = case["kv_heads"], case["head_dim"], case.get("window", 0)
    g = case["heads"] // kvh
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (n, t) in enumerate(zip(_lengths(case), _counts(case))):
        if n and t:
            ends = torch.arange(n - t + 1, n + 1, device="cuda")
            for j in range(kvh):
                if pages_of is None:
                    token = torch.arange(max(0, n - t + 1 - window) if window else 0, n, device="cuda")
                else:
                    chosen = np.asarray([p for p in pages_of[r][j] if p >= 0], dtype=np.int64)
                    token = torch.from_numpy((chosen[:, None] * page + np.arange(page)).ravel()).cuda()
                    token = token[token < n]
                where = state["table"][r].long()[token // page]
                k = state["k_pages"][where, j, token % page].double()
                v = state["v_pages"][where, j, token % page].double()
                hidden = token[None] >= ends[:, None]
                if window:
                    hidden |= token[None] < ends[:, None] - window
                for head in range(j * g, (j + 1) * g):
                    s = (state["q"][at:at + t, head].double() @ k.T) / math.sqrt(d)
                    s[hidden] = -math.inf
                    blank = hidden.all(1)
                    s[blank] = 0.0
                    if case.get("sinks"):
                        s = torch.cat((s, state["sinks"][head].double().expand(t, 1)), 1)
                    p = torch.softmax(s, 1)[:, :len(token)]
                    p[blank] = 0.0
                    out[at:at + t, head] = p @ v
        at += t
    return out


def _exact_select(state):
    case, page = state["case"], state["case"]["page"]
    kvh, d = case["kv_heads"], case["head_dim"]
    selected = np.full(tuple(state["selected"].shape), -1, dtype=np.int32)
    for r, n in enumerate(_lengths(case)):
        pages = -(-n // page)
        if pages == 0:
            continue
        held = state["k_bounds"][state["table"][r, :pages].long()].double()
        for j in range(kvh):
            q = state["q"][r].double().view(kvh, -1, d)[j]
            # the bound as one product: the positive part meets the greatest value, the negative the least
            s = q.clamp_min(0) @ held[:, j, 1].T + q.clamp_max(0) @ held[:, j, 0].T
            s = s.amax(0).cpu().numpy().astype(np.float32)
            forced = set(range(min(case["first"], pages))) | set(range(max(0, pages - case["last"]), pages))
            free = sorted((p for p in range(pages) if p not in forced), key=lambda p: -s[p])
            keep = sorted([*forced, *free[:max(0, case["count"] - len(forced))]])
            selected[r, j, :len(keep)] = keep
    return selected


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(state)
    if case["kind"] == "sparse":
        selected = _exact_select(state)
        return selected, _exact_attention(state, selected)
    return _exact_attention(state)
