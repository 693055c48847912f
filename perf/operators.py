"""The operators of a decode step around its weights: rotary positions, a KV cache of 4 bits
(append, read back, attention with windows) and sampling.

Every case is one pass as a serving program makes it for one layer (or for the head of the
model): ``run`` calls ``HipDecodeBackend`` where ``own`` is true and computes the same formulas
with elementary torch operations where it is false.  ``exact`` restates them in float64.

The cache's layout is written out here once more, by its definition: a group of ``group`` dims of
one token and KV head holds codes c of 0 .. 15 with a step s and a minimum m, value c s + m.
``k_codes`` int32 [B, KVH, capacity, D/8], dim d in nibble d % 8 of word d / 8; ``k_scales`` f16
[B, KVH, capacity, D/group, 2] (s, m); ``v_codes`` int32 [B, KVH, capacity/8, D], token t of a
block of eight in nibble (t >> 1) + 4 (t & 1); ``v_scales`` f16 [B, KVH, capacity/8, D/group, 2, 8].
"""

from __future__ import annotations

import functools
import math

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_MAX_TOKENS = 2 * 131072 * 8 * 128       # sequences x tokens x KV heads x head_dim of the largest cache
_MAX_LOGITS = 64 * 152064


def listed() -> list[dict]:
    return [
        # one token of a 1B model: the smallest call of a decode step
        {"name": "rotary-step", "kind": "rotary", "tokens": 1, "heads": 32, "kv_heads": 8, "head_dim": 64, "rotary": 64,
         "interleaved": False, "far": 575, "factor": 1.0, "dtype": "f16"},
        # a prompt of odd length far into a stretched context, half of the head rotated, interleaved pairs
        {"name": "rotary-prompt", "kind": "rotary", "tokens": 8191, "heads": 64, "kv_heads": 8, "head_dim": 128,
         "rotary": 64, "interleaved": True, "far": 131072, "factor": 32.0, "dtype": "bf16"},
        # one new token for each of eight sequences
        {"name": "cache-step", "kind": "cache", "batch": 8, "tokens": 1, "kv_heads": 8, "head_dim": 64, "group": 32,
         "offset": 1029, "dtype": "f16"},
        # three prompts of unequal length that begin inside a block of the cache
        {"name": "cache-ragged", "kind": "cache", "batch": 3, "tokens": 2731, "kv_heads": 10, "head_dim": 128, "group": 64,
         "offset": 77, "dtype": "bf16"},
        # one long prompt
        {"name": "cache-prompt", "kind": "cache", "batch": 1, "tokens": 16384, "kv_heads": 8, "head_dim": 128, "group": 128,
         "offset": 0, "dtype": "f16"},
        # one layer of the 1B decode: one sequence, a few hundred tokens
        {"name": "attention-step", "kind": "attention", "batch": 1, "length": 575, "heads": 32, "kv_heads": 8,
         "head_dim": 64, "group": 32, "window": 0, "first": 0, "sinks": False, "dtype": "f16"},
        # four sequences of unequal length, 40 query heads on 10 KV heads of dim 128
        {"name": "attention-ragged", "kind": "attention", "batch": 4, "length": 4001, "heads": 40, "kv_heads": 10,
         "head_dim": 128, "group": 64, "window": 0, "first": 0, "sinks": False, "dtype": "bf16"},
        # a window of 128 tokens and four first tokens over long contexts, learned sinks, eight sequences
        {"name": "attention-window", "kind": "attention", "batch": 8, "length": 16385, "heads": 64, "kv_heads": 8,
         "head_dim": 64, "group": 32, "window": 128, "first": 4, "sinks": True, "dtype": "f16"},
        # two sequences at a long context: the largest read
        {"name": "attention-long", "kind": "attention", "batch": 2, "length": 131072, "heads": 64, "kv_heads": 8,
         "head_dim": 128, "group": 128, "window": 0, "first": 0, "sinks": False, "dtype": "bf16"},
        # one sequence, the usual truncations
        {"name": "sample-step", "kind": "sample", "rows": 1, "vocab": 128256, "temperature": 0.7, "top_k": 50,
         "top_p": 0.9, "min_p": 0.0, "masked": False, "dtype": "f16"},
        # eight sequences of a large vocabulary, no top-k, part of the vocabulary masked
        {"name": "sample-min-p", "kind": "sample", "rows": 8, "vocab": 201088, "temperature": 1.0, "top_k": 0,
         "top_p": 1.0, "min_p": 0.02, "masked": True, "dtype": "bf16"},
        # 64 sequences, each with its own settings (greedy and untruncated ones among them), 32-bit logits
        {"name": "sample-batch", "kind": "sample", "rows": 64, "vocab": 152064, "temperature": 1.2, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0, "masked": False, "dtype": "f32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "cache", "attention", "attention", "sample"])
    dtype = rng.choice(["f16", "bf16"])
    head_dim = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 10])
    if kind == "rotary":
        heads = kv_heads * rng.choice([1, 4, 5, 8])
        most = min(32768, 8191 * 72 * 128 // ((heads + kv_heads) * head_dim))
        return {"kind": kind, "tokens": _log_int(rng, 1, most), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary": rng.choice([head_dim // 4, head_dim // 2, head_dim]), "interleaved": rng.random() < 0.5,
                "far": _log_int(rng, 64, 1 << 20), "factor": rng.choice([1.0, 4.0, 8.0, 32.0]),
                "dtype": rng.choice(["f16", "bf16", "f32"])}
    if kind == "cache":
        batch = _log_int(rng, 1, 64)
        most = max(2, 16384 * 8 * 128 // (batch * kv_heads * head_dim))
        return {"kind": kind, "batch": batch, "tokens": _log_int(rng, 1, min(most, 16384)), "kv_heads": kv_heads,
                "head_dim": head_dim, "group": rng.choice([g for g in (32, 64, 128) if g <= head_dim]),
                "offset": rng.randint(0, 4095), "dtype": rng.choice(["f16", "bf16", "f32"])}
    if kind == "attention":
        batch = _log_int(rng, 1, 64)
        most = min(131072, _MAX_TOKENS // (batch * kv_heads * head_dim) // 32 * 32 - 64)
        window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
        return {"kind": kind, "batch": batch, "length": _log_int(rng, 1, most),
                "heads": kv_heads * rng.choice([1, 2, 4, 5, 8, 16]), "kv_heads": kv_heads, "head_dim": head_dim,
                "group": rng.choice([g for g in (32, 64, 128) if g <= head_dim]), "window": window,
                "first": rng.choice([0, 1, 4, 33]) if window else 0, "sinks": rng.random() < 0.4, "dtype": dtype}
    rows = _log_int(rng, 1, 64)
    return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 1000, min(201088, _MAX_LOGITS // rows)),
            "temperature": round(rng.uniform(0.2, 2.0), 2), "top_k": rng.choice([0, 1, _log_int(rng, 2, 1000)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
            "min_p": rng.choice([0.0, round(rng.uniform(0.005, 0.3), 3)]), "masked": rng.random() < 0.3,
            "dtype": rng.choice(["f16", "bf16", "f32"])}


# ------------------------------------------------------------------------------- inputs
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(std)


def _capacity(tokens: int) -> int:
    return -(-tokens // 32) * 32


def _lengths(case: dict) -> list[int]:
    """Unequal lengths, the case's own first and half of it at the end."""
    n, b = case["length"], case["batch"]
    return [max(1, n - n * i // (2 * b)) for i in range(b)]


def _visible(case: dict) -> list[int]:
    w, f = case["window"], case["first"]
    return [n if w == 0 or n <= w + f else w + min(f, n - w) for n in _lengths(case)]


def _step_minimum(x, group):
    """Groups' minimum m, rounded to f16, and step s (seven significant bits, at least 2^-24, 15 s
    at least max - m) of float64 x [..., D]: the group's x and f64 m, s, all with a last axis of it."""
    xg = x.unflatten(-1, (-1, group))
    m = xg.amin(-1, keepdim=True).clamp(-65504.0, 65504.0).to(torch.float16).double()
    reach = (xg.amax(-1, keepdim=True) - m).clamp_min(0.0)
    raw = reach / 15.0
    # 2^e from its bits: a power function may be an ulp off
    lsb = (((torch.frexp(raw).exponent - 7).clamp_min(-24).long() + 1023) << 52).view(torch.float64)
    s = torch.ceil(raw / lsb) * lsb
    return xg, m, s.clamp_max(4352.0)


def _codes(xg, m, s):
    return torch.where(s > 0, torch.round((xg - m) / s.where(s > 0, torch.ones_like(s))).clamp(0, 15), torch.zeros_like(xg))


def _pack_nibbles(codes, dim, order):
    """Eight codes along `dim` (of size 8) into one int32, code i in nibble order[i]."""
    shifts = torch.tensor([4 * o for o in order], device=codes.device)
    shifts = shifts.view([8 if i == dim % codes.dim() else 1 for i in range(codes.dim())])
    words = (codes.to(torch.int64) << shifts).sum(dim)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


_TOKEN_NIBBLE = [(t >> 1) + 4 * (t & 1) for t in range(8)]


def _cache(g, batch, kv_heads, capacity, head_dim, group):
    """A filled cache: K with a spread of channel means, V without.  One head at a time."""
    parts = {"k_codes": [], "k_scales": [], "v_codes": [], "v_scales": []}
    for _ in range(batch * kv_heads):
        k = _normal(g, (capacity, head_dim)).add_(_normal(g, (1, head_dim), 1.5))
        xg, m, s = _step_minimum(k.double(), group)
        parts["k_codes"].append(_pack_nibbles(_codes(xg, m, s).reshape(capacity, head_dim // 8, 8), 2, range(8)))
        parts["k_scales"].append(torch.cat((s, m), -1).to(torch.float16))
        xg, m, s = _step_minimum(_normal(g, (capacity, head_dim)).double(), group)
        parts["v_codes"].append(_pack_nibbles(_codes(xg, m, s).reshape(capacity // 8, 8, head_dim), 1, _TOKEN_NIBBLE))
        sm = torch.cat((s, m), -1).to(torch.float16).unflatten(0, (-1, 8))          # [blocks, 8, groups, 2]
        parts["v_scales"].append(sm.permute(0, 2, 3, 1).contiguous())
    return {n: torch.stack(p).unflatten(0, (batch, kv_heads)) for n, p in parts.items()}


def prepare(case: dict, seed: int) -> dict:
    g, kind, dt = _gen(seed), case["kind"], _DTYPES[case["dtype"]]
    state = {"case": case}
    if kind == "rotary":
        t, r = case["tokens"], case["rotary"]
        state["q"] = _normal(g, (t, case["heads"], case["head_dim"])).to(dt)
        state["k"] = _normal(g, (t, case["kv_heads"], case["head_dim"])).to(dt)
        state["positions"] = torch.arange(t, device="cuda", dtype=torch.int32) + max(0, case["far"] - t)
        # the low frequencies stretched by the factor, the high ones kept: frequencies of a long context
        f = 500000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        keep = torch.linspace(1.0, 0.0, r // 2, device="cuda", dtype=torch.float64)
        state["inv_freq"] = f * keep + f / case["factor"] * (1 - keep)
        state["amplitude"] = 0.1 * math.log(case["factor"]) + 1.0
        state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
    elif kind == "cache":
        b, t, h, d = case["batch"], case["tokens"], case["kv_heads"], case["head_dim"]
        cap, groups = _capacity(case["offset"] + t + 2 * b), d // case["group"]
        state["k"] = _normal(g, (b, t, h, d)).add_(_normal(g, (1, 1, h, d), 1.5)).to(dt)
        state["v"] = _normal(g, (b, t, h, d)).to(dt)
        state["starts"] = torch.arange(b, device="cuda", dtype=torch.int32) * 2 + case["offset"]
        state["cache"] = {
            "k_codes": torch.zeros((b, h, cap, d // 8), device="cuda", dtype=torch.int32),
            "k_scales": torch.zeros((b, h, cap, groups, 2), device="cuda", dtype=torch.float16),
            "v_codes": torch.zeros((b, h, cap // 8, d), device="cuda", dtype=torch.int32),
            "v_scales": torch.zeros((b, h, cap // 8, groups, 2, 8), device="cuda", dtype=torch.float16)}
        state["k_out"], state["v_out"] = torch.empty_like(state["k"]), torch.empty_like(state["v"])
    elif kind == "attention":
        b, h, d = case["batch"], case["heads"], case["head_dim"]
        state["cache"] = _cache(g, b, case["kv_heads"], _capacity(case["length"] + 1), d, case["group"])
        state["q"] = _normal(g, (b, h, d)).to(dt)
        state["lengths"] = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        state["sinks"] = _normal(g, (h,)).to(dt) if case["sinks"] else None
        state["out"] = torch.empty_like(state["q"])
    else:
        m, v = case["rows"], case["vocab"]
        # a bulk of small logits and a thin upper tail, as language models leave them; some rows sharper
        x = _normal(g, (m, v), 1.6)
        x += torch.empty((m, v), device="cuda").exponential_(0.8, generator=g)
        x *= torch.linspace(0.8, 1.6, m, device="cuda")[:, None]
        if case["masked"]:
            x = x.masked_fill(torch.rand((m, v), generator=g, device="cuda") < 0.4, -math.inf)
        state["logits"] = x.to(dt)
        state["uniforms"] = torch.rand(m, generator=g, device="cuda")
        row = torch.arange(m, device="cuda")
        # a few rows greedy, a few without truncation, as requests of one batch differ
        state["temperature"] = torch.where(row % 16 == 5, 0.0, case["temperature"]).float()
        state["top_k"] = torch.where(row % 16 == 9, 0, case["top_k"]).to(torch.int32)
        state["top_p"] = torch.where(row % 16 == 9, 1.0, case["top_p"]).float()
        state["min_p"] = torch.full((m,), case["min_p"], device="cuda")
        state["tokens"] = torch.empty(m, device="cuda", dtype=torch.int64)
        state["probs"] = torch.empty(m, device="cuda")
    return state


# ------------------------------------------------------------------------------- the framework's calls
@functools.lru_cache(maxsize=None)
def _backend():
    from thintensor_amd.backend import HipDecodeBackend

    return HipDecodeBackend(torch.device("cuda:0"), torch.float16, 2048, 2048, 512, 8192)


def _own_cache(state):
    if "handle" not in state:                 # the object that a program makes once around a cache's tensors
        from thintensor_amd.kv_cache import Int4KvCache

        c = state["cache"]
        state["handle"] = Int4KvCache(c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"])
    return state["handle"]


def _run_own(state):
    case, be = state["case"], _backend()
    if case["kind"] == "rotary":
        be.rotary_rows(state["q"], state["k"], state["positions"], state["inv_freq"], state["q_out"], state["k_out"],
                       interleaved=case["interleaved"], amplitude=state["amplitude"])
        return state["q_out"], state["k_out"]
    if case["kind"] == "cache":
        cache = _own_cache(state)
        be.kv_append_int4(cache, state["k"], state["v"], state["starts"])
        be.kv_read_int4(cache, state["k_out"], state["v_out"], state["starts"])
        return state["k_out"], state["v_out"]
    if case["kind"] == "attention":
        return be.gqa_attention_int4(state["q"], _own_cache(state), state["out"], state["lengths"],
                                     window=case["window"], first_tokens=case["first"], sinks=state["sinks"])
    be.sample_rows(state["logits"], state["uniforms"], state["tokens"], temperature=state["temperature"],
                   top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"], probs=state["probs"])
    return state["tokens"], state["probs"]


# ------------------------------------------------------------------------------- the plain forms
def _rotate(x, cos, sin, rotary, interleaved):
    head, rest = x[..., :rotary].float(), x[..., rotary:].float()
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : rotary // 2], head[..., rotary // 2:])
    c, s = cos[:, None], sin[:, None]
    first, second = a * c - b * s, b * c + a * s
    head = torch.stack((first, second), -1).flatten(-2) if interleaved else torch.cat((first, second), -1)
    return torch.cat((head, rest), -1).to(x.dtype)


def _plain_rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["inv_freq"]
    cos, sin = (angle.cos() * state["amplitude"]).float(), (angle.sin() * state["amplitude"]).float()
    return tuple(_rotate(state[n], cos, sin, case["rotary"], case["interleaved"]) for n in ("q", "k"))


def _plain_cache(x, group):
    # codes in 64 bits: they lie on borders between two codes otherwise
    xg, m, s = _step_minimum(x.double(), group)
    return (_codes(xg, m, s) * s + m).flatten(-2).to(x.dtype)


def _plain_tokens(state):
    """The cache's tokens that some query may see: K and V [B, KVH, N, D] in 32 bits and which of the
    N count for which sequence."""
    case, c, lengths = state["case"], state["cache"], state["lengths"].long()
    capacity, window, first = c["k_codes"].shape[2], case["window"], case["first"]
    at = torch.arange(capacity, device="cuda")
    shifts = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    if window and window + first + 8 < capacity:
        # whole blocks of eight tokens around the window and the first tokens
        blocks = torch.cat((torch.arange(-(-first // 8), device="cuda").expand(len(lengths), -1),
                            (lengths[:, None] - window).clamp_min(0) // 8 + torch.arange(window // 8 + 2, device="cuda")), 1)
        seen = torch.arange(blocks.shape[1], device="cuda") >= -(-first // 8)
        inside = blocks < capacity // 8
        blocks = blocks.clamp_max(capacity // 8 - 1)
        at = (blocks[..., None] * 8 + torch.arange(8, device="cuda")).flatten(1)                  # [B, N]
        start = (lengths - window)[:, None]
        counts = torch.where(seen.repeat_interleave(8), (at >= start) & (at < lengths[:, None]),
                             (at < first) & (at < start))
        counts &= inside.repeat_interleave(8, 1)
        b = torch.arange(len(lengths), device="cuda")[:, None]
        kc, ks = c["k_codes"].transpose(1, 2)[b, at].transpose(1, 2), c["k_scales"].transpose(1, 2)[b, at].transpose(1, 2)
        vc = c["v_codes"].transpose(1, 2)[b, blocks].transpose(1, 2)
        vs = c["v_scales"].transpose(1, 2)[b, blocks].transpose(1, 2)
    else:
        at = at[None]
        counts = at < lengths[:, None]
        if window:
            counts = counts & ((at >= lengths[:, None] - window) | (at < first))
        kc, ks, vc, vs = c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"]
    group = case["group"]
    k = ((kc[..., None] >> shifts) & 15).flatten(-2).unflatten(-1, (-1, group)).float()
    k = (k * ks[..., :1].float() + ks[..., 1:].float()).flatten(-2)
    nib = torch.tensor(_TOKEN_NIBBLE, device="cuda", dtype=torch.int32)[:, None] * 4
    v = ((vc[..., None, :] >> nib) & 15).unflatten(-1, (-1, group)).float()                         # [B, H, blocks, 8, G, g]
    sm = vs.permute(0, 1, 2, 4, 5, 3).float()[..., None]                                          # [B, H, blocks, 2, 8, G, 1]
    v = (v * sm[:, :, :, 0] + sm[:, :, :, 1]).flatten(-2).flatten(2, 3)
    return k, v, counts


def _plain_attention(state):
    case, q = state["case"], state["q"]
    b, h, d = q.shape
    k, v, counts = _plain_tokens(state)
    qg = q.float().view(b, case["kv_heads"], h // case["kv_heads"], d)
    s = torch.matmul(k, qg.transpose(2, 3).contiguous()) * d ** -0.5                              # [B, KVH, N, G]
    s = s.masked_fill(~counts[:, None, :, None], -math.inf)
    top = s.amax(2, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].float().view(1, case["kv_heads"], 1, -1)
        top = torch.maximum(top, sink)
    p = torch.exp(s - top)
    total = p.sum(2, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.matmul(p.transpose(2, 3).contiguous(), v) / total.transpose(2, 3)
    return out.reshape(b, h, d).to(q.dtype)


def _plain_sample(state):
    # 64 bits: a cumulative sum over the vocabulary is compared with a border
    x, t = state["logits"], state["temperature"].double()[:, None]
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    xs = xs.double()
    top, live = xs[:, :1], xs > -math.inf
    z = torch.where(t > 0, (top - xs) / t.where(t > 0, torch.ones_like(t)), torch.where(xs == top, 0.0, math.inf))
    w = torch.where(live, torch.exp(-z), 0.0)
    cum = w.cumsum(-1)
    n = live.sum(-1)
    k = torch.where(state["top_k"] > 0, torch.minimum(state["top_k"].long(), n), n)
    k = torch.where(t[:, 0] > 0, k, 1)
    mass = cum.gather(1, k[:, None] - 1)
    p = state["top_p"].double()[:, None]
    n_p = torch.where(state["top_p"] < 1, (cum < p * mass).sum(-1) + 1, k)
    n_m = (w >= state["min_p"].double()[:, None]).sum(-1).clamp_min(1)
    n = torch.minimum(torch.minimum(k, n_p), torch.where(state["min_p"] > 0, n_m, k))
    kept = cum.gather(1, n[:, None] - 1)
    j = torch.minimum((cum <= state["uniforms"].double()[:, None] * kept).sum(-1), n - 1)[:, None]
    return order.gather(1, j)[:, 0], (w.gather(1, j) / kept)[:, 0].float()


def run(state: dict):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "rotary":
        return _plain_rotary(state)
    if kind == "cache":
        return tuple(_plain_cache(state[n], state["case"]["group"]) for n in ("k", "v"))
    return _plain_attention(state) if kind == "attention" else _plain_sample(state)


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rotary":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["head_dim"] * size + 4 * case["tokens"] + 4 * case["rotary"], "flops": 3 * n * case["rotary"]}
    if case["kind"] == "cache":
        n = case["batch"] * case["tokens"] * case["kv_heads"]
        packed = case["head_dim"] + 8 * case["head_dim"] // case["group"]
        return {"bytes": n * (4 * case["head_dim"] * size + 2 * packed), "flops": n * case["head_dim"] * 10}
    if case["kind"] == "attention":
        d, visible = case["head_dim"], sum(_visible(case))
        io = 2 * case["batch"] * case["heads"] * d * size
        return {"bytes": visible * case["kv_heads"] * (d + 8 * d // case["group"]) + io, "flops": 4 * visible * case["heads"] * d}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + 32 * case["rows"], "flops": 4 * n}


# ------------------------------------------------------------------------------- float64, from the definitions
def _exact_rotary(state):
    case = state["case"]
    turn = torch.polar(torch.tensor(state["amplitude"], dtype=torch.float64, device="cuda"),
                       state["positions"].double()[:, None] * state["inv_freq"])[:, None]
    outs = []
    for x in (state["q"].double(), state["k"].double()):
        out, r = x.clone(), case["rotary"]
        pairs = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
        z = torch.complex(x[..., pairs[0]], x[..., pairs[1]]) * turn
        out[..., pairs[0]], out[..., pairs[1]] = z.real, z.imag
        outs.append(out)
    return tuple(outs)


def _exact_cache(x, group):
    a = x.double().cpu().numpy()
    a = a.reshape(-1, group)
    m = a.min(1).astype(np.float16).astype(np.float64)
    reach = np.maximum(a.max(1) - m, 0.0)
    # the grid of seven significant bits: an integer of at most 128 times a power of two
    e = np.maximum(np.where(reach > 0, np.floor(np.log2(np.maximum(reach, 1e-300) / 15.0)), 0) - 8, -24)
    while True:
        n = np.ceil(reach / (15.0 * np.exp2(e)))
        wide = n > 128
        if not wide.any():
            break
        e[wide] += 1
    s = n * np.exp2(e)
    codes = np.rint(np.divide(a - m[:, None], s[:, None], out=np.zeros_like(a), where=s[:, None] > 0)).clip(0, 15)
    return (codes * s[:, None] + m[:, None]).reshape(x.shape)


def _exact_attention(state):
    case, c, lengths = state["case"], state["cache"], _lengths(state["case"])
    b, h, d = state["q"].shape
    per, group = h // case["kv_heads"], case["group"]
    out = torch.zeros((b, h, d), dtype=torch.float64, device="cuda")
    for i in range(b):
        n = lengths[i]
        t = torch.arange(n, device="cuda")
        if case["window"]:
            t = t[(t < case["first"]) | (t >= n - case["window"])]
        for j in range(case["kv_heads"]):
            words = c["k_codes"][i, j][t].long() & 0xffffffff
            k = torch.stack([(words >> (4 * a)) & 15 for a in range(8)], -1).reshape(len(t), d).double()
            sm = c["k_scales"][i, j][t].double().repeat_interleave(group, 1)
            k = k * sm[..., 0] + sm[..., 1]
            nib = (((t % 8) >> 1) + 4 * (t % 2)) * 4
            v = (((c["v_codes"][i, j][t // 8].long() & 0xffffffff) >> nib[:, None]) & 15).double()
            vs = c["v_scales"][i, j][t // 8, :, :, t % 8].double().repeat_interleave(group, 1)
            v = v * vs[..., 0] + vs[..., 1]
            for g in range(j * per, (j + 1) * per):
                s = (k * state["q"][i, g].double()).sum(1) / math.sqrt(d)
                if state["sinks"] is not None:
                    s = torch.cat((s, state["sinks"][g].double()[None]))
                p = torch.softmax(s, 0)[: len(t)]
                out[i, g] = (p[:, None] * v).sum(0)
    return out


def _exact_sample(state):
    tokens, probs = [], []
    for i in range(state["case"]["rows"]):
        x = state["logits"][i].double().cpu().numpy()
        t, k, p, mp, u = (float(state[n][i]) for n in ("temperature", "top_k", "top_p", "min_p", "uniforms"))
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -math.inf]
        if t <= 0:
            order = order[:1]
        w = np.exp((x[order] - x[order[0]]) / t) if t > 0 else np.ones(1)
        w = w[: int(k)] if k > 0 else w
        if p < 1:
            w = w[: 1 + int(np.searchsorted(np.cumsum(w), p * np.sum(w)))]
        w = w[: max(1, int(np.count_nonzero(w >= mp)))]
        cum = np.cumsum(w)
        j = min(int(np.searchsorted(cum, u * cum[-1], side="right")), len(w) - 1)
        tokens.append(int(order[j]))
        probs.append(w[j] / cum[-1])
    return np.array(tokens), np.array(probs)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(state)
    if case["kind"] == "cache":
        return tuple(_exact_cache(state[n], case["group"]) for n in ("k", "v"))
    return _exact_attention(state) if case["kind"] == "attention" else _exact_sample(state)
