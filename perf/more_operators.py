"""Operators for caches that hold long requests in less memory, one dict per timed case.

``store`` writes new tokens into a cache of 4-bit keys and values (their norm and
rotation in the same pass) and reads the cache back in 16 bits; ``decode`` is the
attention of new tokens over such a cache; ``weigh`` adds up the attention that every
cached key receives; ``evict`` keeps the rows of a cache that received most of it.
``own`` selects the package's kernels; without it the same is computed by elementary
torch operations in 32 bits.

A 4-bit row holds groups of 32 columns (the last one filled up with zeros) with a float16
scale d each; a column is d * (n - 8) for its code n = 0 .. 15.  d is the group's value of
largest magnitude over -8.  Eight codes make a word of 32 bits, the first in its lowest
bits: word 4 g + o of a value row holds columns 32 g + 8 o and on, word o * groups + g of
a key row.

Run from the repository's root, which holds the package folder.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def _store(B, T, S, H, Hk, D, dtype, R, interleaved=False):
    return {"op": "store", "B": B, "T": T, "S": S, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "R": R,
            "interleaved": interleaved}


def _decode(B, T, S, H, Hk, D, dtype, left, sinks):
    return {"op": "decode", "B": B, "T": T, "S": S, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "left": left, "sinks": sinks}


def _weigh(B, T, S, H, Hk, D, dtype, left, sinks, q4=False):
    return {"op": "weigh", "B": B, "T": T, "S": S, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "left": left, "sinks": sinks,
            "q4": q4}


def _evict(B, S, Hk, D, dtype, budget, recent, sinks, q4=False, out=False):
    return {"op": "evict", "B": B, "S": S, "Hk": Hk, "D": D, "dtype": dtype, "budget": budget, "recent": recent,
            "sinks": sinks, "q4": q4, "out": out}


def listed():
    return [
        # The smallest call: one new token of one request, and its short cache back.
        {"name": "store_1", **_store(1, 1, 256, 8, 8, 64, "fp16", 64)},
        # A whole prompt at the benchmark's length, grouped K/V heads.
        {"name": "store_prompt", **_store(1, 32768, 32768, 32, 8, 128, "bf16", 128)},
        # Prompts of a ragged batch: D = 80 (a half-filled group), part of the head turned, neighbouring pairs.
        {"name": "store_ragged", **_store(3, 1777, 2000, 12, 4, 80, "fp16", 32, interleaved=True)},
        # One request's next token over a 4096-token window: too few rows to fill the card.
        {"name": "decode_1", **_decode(1, 1, 8192, 32, 8, 128, "bf16", 4095, 4)},
        # The next tokens of a large batch of ragged requests, every cached token seen.
        {"name": "decode_128", **_decode(128, 1, 8192, 32, 8, 128, "bf16", 8192, 0)},
        # Wide heads, eight query heads on each K/V head, two drafted tokens: more rows than a matrix tile.
        {"name": "decode_wide", **_decode(4, 3, 5000, 16, 2, 256, "fp16", 2000, 16)},
        # The weights of a serving batch's step.
        {"name": "weigh_step", **_weigh(64, 1, 8192, 32, 8, 128, "bf16", 8192, 0)},
        # The weights of a whole prompt.
        {"name": "weigh_prompt", **_weigh(1, 8192, 8192, 32, 8, 128, "bf16", 8192, 0)},
        # The weights that the last tokens of a long prompt give to its 4-bit keys.
        {"name": "weigh_q4", **_weigh(2, 32, 32768, 16, 4, 64, "fp16", 32768, 0, q4=True)},
        # Half of every cache of a batch goes, in place.
        {"name": "evict_batch", **_evict(16, 8192, 8, 128, "bf16", 4096, 512, 4)},
        # The same of a larger batch of 4-bit caches, three quarters.
        {"name": "evict_q4", **_evict(64, 16384, 8, 128, "bf16", 4096, 256, 4, q4=True)},
        # What is kept of one long prompt moves into a small cache.
        {"name": "evict_prompt", **_evict(1, 32768, 8, 128, "bf16", 2048, 64, 4, out=True)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes over the listed cases' ranges, odd ones among them, none dearer than the largest listed case of its kind."""
    while True:
        op = rng.choice(["store", "decode", "decode", "weigh", "weigh", "evict"])
        dtype = rng.choice(["bf16", "fp16"])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        H = rng.choice([2, 4, 8, 12, 16, 32])
        Hk = H // rng.choice([g for g in (1, 2, 3, 4, 8) if H % g == 0])
        B, S = _log(rng, 1, 128), _log(rng, 64, 32768)
        if op == "store":
            T = rng.choice([1, 1, 2, 5, S, S, rng.randint(1, S)])
            if B * S * Hk * D > 32768 * 8 * 128 or B * T * (H + 2 * Hk) * D > 32768 * 48 * 128:
                continue
            return _store(B, T, S, H, Hk, D, dtype, rng.choice([D, D, 32]), rng.random() < 0.4)
        if op == "decode":
            left = rng.choice([S, S, _log(rng, 16, 8192) - 1])
            if B * S * Hk * D > 128 * 8192 * 8 * 128:
                continue
            return _decode(B, rng.choice([1, 1, 1, 2, 3, 5]), S, H, Hk, D, dtype, left, rng.choice([0, 0, 1, 4, 16, 100]))
        if op == "weigh":
            T = rng.choice([1, 1, 2, 16, 32, 100, S])
            left = rng.choice([S, S, S, _log(rng, 16, 8192) - 1])
            if T > S or B * S * Hk * D > 64 * 8192 * 8 * 128 or B * H * T * S * max(D, 64) > 32 * 8192 * 8192 * 128:
                continue
            return _weigh(B, T, S, H, Hk, D, dtype, left, rng.choice([0, 0, 4, 16]), rng.random() < 0.4)
        q4 = rng.random() < 0.5
        budget = max(8, int(S * rng.uniform(0.1, 0.9)))
        recent, sinks = rng.randint(0, budget // 2), rng.choice([0, 1, 4, 4])
        if B * S * Hk * D > (4 if q4 else 1) * 16 * 8192 * 8 * 128 or recent + sinks > budget or budget > S:
            continue
        return _evict(B, S, Hk, D, dtype, budget, recent, sinks, q4, rng.random() < 0.3)


# ---------------------------------------------------------------- inputs


def _lens(gen, B, S, least):
    """Lengths of a batch: from half of the room to all of it, the first request full."""
    n = (torch.rand(B, generator=gen, device="cuda") * (S // 2 + 1)).int() + (S - S // 2)
    n[0] = S
    return n.clamp_(min=least, max=S)


def _tables(P, R):
    """cos and sin of the angles of positions 0 .. P - 1 (formed in 64 bits, kept in 32)."""
    inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    a = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _first_lse(s, c):
    """What the attention itself left of its softmax: the rows' log-sums."""
    B, T, S, H, Hk, D = (c[n] for n in ("B", "T", "S", "H", "Hk", "D"))
    k = _columns(s["cache"][0], True, s["cache"][1], D) if c["q4"] else s["k_cache"].view(B, S, Hk, D).transpose(1, 2).float()
    q = _split_rows(s["q"], Hk, D)
    lse = torch.empty(B, Hk, q.shape[2], device="cuda")
    step = max(1, (1 << 29) // S)
    for b in range(B):
        for h in range(Hk):
            for r in range(0, q.shape[2], step):
                seen = _seen(s["lens"][b:b + 1], c, H // Hk)[0, r:r + step]
                x = (q[b, h, r:r + step] @ k[b, h].T * D ** -0.5).masked_fill_(~seen, -math.inf)
                lse[b, h, r:r + step] = torch.logsumexp(x, -1)
    return lse.view(B, Hk, T, H // Hk).transpose(2, 3).reshape(B, H, T)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, S, Hk, D = c["B"], c["S"], c["Hk"], c["D"]

    def x(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    def rows():  # keys (or values) of a whole 4-bit cache
        return x(B, Hk, S, D)

    s = {"case": c}
    if c["op"] == "store":
        T, H, groups = c["T"], c["H"], -(-D // 32)
        s["q"], s["k"], s["v"] = x(B, T, H * D), x(B, T, Hk * D), x(B, T, Hk * D)
        s["qw"], s["kw"] = (1 + 0.1 * torch.randn(D, generator=gen, device="cuda") for _ in range(2))
        s["cos"], s["sin"] = _tables(S, c["R"])
        s["lens"] = _lens(gen, B, S, T)
        s["cache"] = tuple(torch.zeros(B, Hk, S, n, device="cuda", dtype=t)
                           for n, t in ((16 * groups, torch.uint8), (groups, torch.float16)) * 2)
    elif c["op"] == "evict":
        s["lens"] = _lens(gen, B, S, 1)
        # a few keys draw most of the attention, some none at all
        w = torch.randn(B, Hk, S, generator=gen, device="cuda").mul_(2).exp_()
        w[torch.rand(B, Hk, S, generator=gen, device="cuda") < 0.1] = 0
        s["seen"] = w.masked_fill_(torch.arange(S, device="cuda") >= s["lens"][:, None, None], 0)
        s["weights"] = w.clone()
        s["cache"] = _packed(rows(), True) + _packed(rows(), False) if c["q4"] else (x(B, S, Hk * D), x(B, S, Hk * D))
        if c["out"]:
            s["to"] = tuple(torch.zeros_like(t[:, :, :c["budget"]] if c["q4"] else t[:, :c["budget"]]).contiguous()
                            for t in s["cache"])
            s["to_weights"] = torch.zeros(B, Hk, c["budget"], device="cuda")
    else:
        T = c["T"]
        s["q"] = x(B, T, c["H"] * D)
        s["lens"] = _lens(gen, B, S, T)
        if c["op"] == "decode":
            s["cache"] = _packed(rows(), True) + _packed(rows(), False)
        else:
            if c["q4"]:
                s["cache"] = _packed(rows(), True) * 2  # values are not looked at
            else:
                s["k_cache"] = x(B, S, Hk * D)
            s["lse"] = _first_lse(s, c)
            s["weights"] = torch.zeros(B, Hk, S, device="cuda")
    if own:
        _package()
    return s


# ---------------------------------------------------------------- the package's calls


def _package():
    path = os.path.abspath("flash-topk-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_topk_attn_v2 as fta

    return fta


def _run_own(s):
    fta = _package()
    c = s["case"]
    Hk = c["Hk"]
    if c["op"] == "store":
        cache = fta.Q4Cache(*s["cache"])
        q = fta.flash_qk_norm_rope_append_q4(s["q"], s["k"], s["v"], cache, s["lens"], c["H"], s["cos"], s["sin"], s["qw"],
                                             s["kw"], eps=EPS, num_kv_heads=Hk, interleaved=c["interleaved"])
        k, v = fta.flash_q4_cache_read(cache, c["D"], s["q"].dtype)
        return {"q": q, "k": k, "v": v}
    if c["op"] == "decode":
        o, lse = fta.flash_window_attn_decode_q4(s["q"], fta.Q4Cache(*s["cache"]), s["lens"], c["H"], c["left"], c["sinks"],
                                                 num_kv_heads=Hk)
        return {"o": o, "lse": lse}
    if c["op"] == "weigh":
        s["weights"].zero_()
        cache = fta.Q4Cache(*s["cache"]) if c["q4"] else s["k_cache"]
        return fta.flash_cache_weights(s["q"], cache, s["lse"], s["lens"], s["weights"], c["H"], c["left"], c["sinks"],
                                       num_kv_heads=Hk)
    s["weights"].copy_(s["seen"])  # the same share of every cache goes each time
    cache, to = s["cache"], s.get("to")
    if c["q4"]:
        cache, to = fta.Q4Cache(*cache), None if to is None else fta.Q4Cache(*to)
    lens, kept = fta.flash_cache_evict(cache, s["weights"], s["lens"], c["budget"], c["recent"], c["sinks"],
                                       out=None if to is None else (to, s["to_weights"]))
    return {"lens": lens, "kept": kept, "cache": s["cache"] if to is None else s["to"],
            "weights": s["weights"] if to is None else s["to_weights"]}


# ---------------------------------------------------------------- the plain forms


def _codes(x):
    """Scales [..., groups] (float16) and codes [..., groups, 32] of rows [..., D] of 16-bit values."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    d = (torch.where(-lo >= hi, lo, hi) / -8).clamp_(-65504, 65504).half()
    n = torch.where(d[..., None] == 0, 8.0, (x / d[..., None].float()).round_() + 8).clamp_(0, 15)
    return d, n.to(torch.uint8)


def _packed(x, key):
    """(codes, scales) as the cache holds them."""
    d, n = _codes(x)
    n = n.unflatten(-1, (4, 8))
    n = (n.transpose(-2, -3) if key else n).flatten(-3)
    return (n[..., 0::2] | n[..., 1::2] << 4), d


def _columns(codes, key, scales, D):
    """The float32 values of a cache's rows [..., D]."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    groups = scales.shape[-1]
    n = n.unflatten(-1, (4, groups, 8)).transpose(-2, -3) if key else n.unflatten(-1, (groups, 4, 8))
    return ((n.flatten(-2).float() - 8) * scales.float()[..., None]).flatten(-2)[..., :D]


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] columns of x turned pair by pair."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, x[..., R:]), -1)


def _norm_rope(x, heads, w, cos, sin, interleaved):
    x = x.float().unflatten(-1, (heads, -1))
    return _rotate(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w, cos, sin, interleaved)


def _plain_store(s, c):
    T, Hk, D, dt = c["T"], c["Hk"], c["D"], s["q"].dtype
    at = s["lens"].long()[:, None] - T + torch.arange(T, device="cuda")
    t = (s["cos"][at][:, :, None], s["sin"][at][:, :, None], c["interleaved"])
    q = _norm_rope(s["q"], c["H"], s["qw"], *t).flatten(-2).to(dt)
    new = _packed(_norm_rope(s["k"], Hk, s["kw"], *t).to(dt), True) + _packed(s["v"].unflatten(-1, (Hk, D)), False)
    row = torch.arange(c["B"], device="cuda")[:, None]
    kc, ks, vc, vs = s["cache"]
    kc[row, :, at], ks[row, :, at], vc[row, :, at], vs[row, :, at] = new
    k, v = _columns(kc, True, ks, D), _columns(vc, False, vs, D)
    return {"q": q, "k": k.to(dt).transpose(1, 2).flatten(-2), "v": v.to(dt).transpose(1, 2).flatten(-2)}


def _split_rows(x, Hk, D):
    """[B, T, H * D] -> [B, Hk, T * G, D]"""
    B, T = x.shape[:2]
    return x.float().view(B, T, Hk, -1, D).transpose(1, 2).reshape(B, Hk, -1, D)


def _seen(lens, c, G):
    """[B, T * G, S]: which cached keys a row sees."""
    T, S = c["T"], c["S"]
    pos = (lens.long()[:, None] - T + torch.arange(T, device="cuda"))[:, :, None]
    j = torch.arange(S, device="cuda")
    return ((j <= pos) & ((j >= pos - c["left"]) | (j < c["sinks"]))).repeat_interleave(G, 1)


def _plain_decode(s, c):
    B, T, H, Hk, D = c["B"], c["T"], c["H"], c["Hk"], c["D"]
    kc, ks, vc, vs = s["cache"]
    x = _split_rows(s["q"], Hk, D) @ _columns(kc, True, ks, D).mT * D ** -0.5
    x = x.masked_fill_(~_seen(s["lens"], c, H // Hk)[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
    l = p.sum(-1, keepdim=True)
    o = (p @ _columns(vc, False, vs, D) / l.clamp(min=1e-30)).view(B, Hk, T, H // Hk, D).transpose(1, 2).reshape(B, T, H * D)
    return {"o": o.to(s["q"].dtype), "lse": (m + torch.log(l)).view(B, Hk, T, H // Hk).transpose(2, 3).reshape(B, H, T)}


def _plain_weigh(s, c):
    B, T, S, H, Hk, D = (c[n] for n in ("B", "T", "S", "H", "Hk", "D"))
    k = _columns(s["cache"][0], True, s["cache"][1], D) if c["q4"] else s["k_cache"].view(B, S, Hk, D).transpose(1, 2).float()
    lse = s["lse"].view(B, Hk, H // Hk, T).transpose(2, 3).reshape(B, Hk, -1, 1)
    x = (_split_rows(s["q"], Hk, D) @ k.mT).mul_(D ** -0.5).sub_(lse)
    s["weights"].zero_()
    return s["weights"].add_(x.exp_().masked_fill_(~_seen(s["lens"], c, H // Hk)[:, None], 0).sum(2))


def _plain_evict(s, c):
    B, S, Hk, budget = c["B"], c["S"], c["Hk"], c["budget"]
    s["weights"].copy_(s["seen"])
    w, lens = s["weights"], s["lens"].long()[:, None, None]
    j = torch.arange(S, device="cuda")
    safe = (j < c["sinks"]) | (j >= lens - c["recent"])
    x = torch.where(j >= lens, -math.inf, torch.where(safe, math.inf, w))
    first = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :budget]  # ties: the lower row first
    new = lens.clamp(max=budget)
    row = torch.arange(budget, device="cuda")
    first = torch.where(row < new, first, S).sort(-1).values  # rows keep their order
    live, at = row < new, first.clamp(max=S - 1)
    kept_w = torch.where(live, w.gather(2, at), 0.0)
    kept = torch.where(live, first, -1).int()

    def rows(x):  # [B, Hk, S, *] of either layout
        return x if c["q4"] else x.view(B, x.shape[1], Hk, -1).transpose(1, 2)

    for x, y in zip(s["cache"], s["to"] if c["out"] else s["cache"]):
        x, y = rows(x), rows(y)[:, :, :budget]
        y.copy_(torch.where(live[..., None], x.gather(2, at[..., None].expand(-1, -1, -1, x.shape[-1])), y))
    if c["out"]:
        s["to_weights"].copy_(kept_w)
    else:
        w.masked_fill_(j < lens, 0.0)
        w[..., :budget] += kept_w
    return {"lens": new.view(B).int(), "kept": kept, "cache": s["to"] if c["out"] else s["cache"],
            "weights": s["to_weights"] if c["out"] else w}


PLAIN = {"store": _plain_store, "decode": _plain_decode, "weigh": _plain_weigh, "evict": _plain_evict}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state, state["case"])


# ---------------------------------------------------------------- work


def _pairs(n, T, left, sinks):
    """Visible (token, key) pairs of one head: the last T of n tokens."""
    t = torch.arange(n - T, n, dtype=torch.float64)
    return float(((t - left).clamp(min=0) * -1 + t + 1 + (t - left).clamp(min=0, max=sinks)).sum())


def work(case):
    c = case
    B, S, Hk, D = c["B"], c["S"], c["Hk"], c["D"]
    row = -(-D // 32) * 18  # bytes of a 4-bit row: codes and scales
    tokens = S if B == 1 else S * (1 + 0.75 * (B - 1)) / B  # the mean length
    if c["op"] == "store":
        n = B * c["T"]
        return {"bytes": int(2 * n * (2 * c["H"] + 2 * Hk) * D + 4 * n * c["R"] + 2 * n * Hk * row + 2 * B * S * Hk * (row + 2 * D)),
                "flops": 8 * n * (c["H"] + Hk) * D}
    if c["op"] == "evict":
        kept = min(c["budget"], tokens)
        moved = 2 * (row if c["q4"] else 2 * D)
        return {"bytes": int(B * Hk * (4 * tokens + 8 * kept + 2 * kept * moved)), "flops": 0}
    T, H = c["T"], c["H"]
    n = int(tokens)
    pairs = B * H * _pairs(n, min(T, n), c["left"], c["sinks"])
    keys = B * Hk * min(n, c["left"] + T + c["sinks"])
    if c["op"] == "decode":
        return {"bytes": int(2 * keys * row + 4 * B * T * H * D + 4 * B * T * H), "flops": 4 * D * pairs}
    return {"bytes": int(keys * (row if c["q4"] else 2 * D) + 2 * B * T * H * D + 4 * B * T * H + 8 * keys), "flops": 2 * D * pairs}


# ---------------------------------------------------------------- the same in 64 bits


def _exact_turned(x, heads, w, c, pos):
    """Norm, weight and rotation in float64; the rotation as a product of complex numbers."""
    x = x.view(*x.shape[:2], heads, c["D"])
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    R = c["R"]
    inv = 10000.0 ** (-torch.arange(0, R, 2, device=x.device, dtype=torch.float64) / R)
    turn = torch.polar(torch.ones((), device=x.device, dtype=torch.float64), pos.double()[..., None, None] * inv)
    head, rest = x[..., :R], x[..., R:]
    if not c["interleaved"]:
        head = head.unflatten(-1, (2, R // 2)).transpose(-1, -2).flatten(-2)
    z = torch.view_as_real(torch.view_as_complex(head.unflatten(-1, (R // 2, 2)).contiguous()) * turn)
    z = (z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    return torch.cat((z, rest), -1)


def _exact_stored(x):
    """What 4 bits keep of rows [..., D] of 16-bit values, group by group, in float64."""
    y = torch.empty(x.shape, device=x.device, dtype=torch.float64)
    for g in range(0, x.shape[-1], 32):
        part = x[..., g:g + 32].double()
        top, low = part.max(-1).values, part.min(-1).values
        d = (-torch.where(top > -low, top, low) / 8).clamp(-65504, 65504).to(torch.float16).double()[..., None]
        n = torch.nan_to_num(torch.round(part / d), nan=0.0, posinf=0.0, neginf=0.0)
        y[..., g:g + 32] = torch.minimum(torch.maximum(n, n.new_tensor(-8)), n.new_tensor(7)) * d
    return y


def _exact_rows(codes, scales, key, D):
    """A cache's rows in float64, word by word."""
    words = codes.contiguous().view(torch.int32).long()
    groups = scales.shape[-1]
    out = torch.empty(*codes.shape[:-1], 32 * groups, device=codes.device, dtype=torch.float64)
    for g in range(groups):
        for o in range(4):
            word = words[..., o * groups + g if key else 4 * g + o]
            for i in range(8):
                out[..., 32 * g + 8 * o + i] = ((word >> (4 * i) & 15) - 8) * scales[..., g].double()
    return out[..., :D]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, S, Hk, D = c["B"], c["S"], c["Hk"], c["D"]
    dt = DTYPES[c["dtype"]]
    if c["op"] == "evict":  # rows are moved, nothing is computed
        return None
    T, H = c["T"], c["H"]
    G, lens = H // Hk, s["lens"].tolist()
    if c["op"] == "store":
        pos = s["lens"].long()[:, None] - T + torch.arange(T, device="cuda")
        out = {"q": _exact_turned(s["q"].double(), H, s["qw"].double(), c, pos).flatten(-2)}
        new = {"k": _exact_stored(_exact_turned(s["k"].double(), Hk, s["kw"].double(), c, pos).to(dt)),
               "v": _exact_stored(s["v"].view(B, T, Hk, D))}
        for n, x in new.items():
            out[n] = torch.zeros(B, S, Hk * D, device="cuda", dtype=torch.float64)
            for b in range(B):
                out[n][b, lens[b] - T:lens[b]] = x[b].flatten(-2)
        return out
    f64 = dict(device="cuda", dtype=torch.float64)
    weights = torch.zeros(B, Hk, S, **f64)
    o, lse = torch.zeros(B, T, H, D, **f64), torch.full((B, H, T), -math.inf, **f64)
    q = s["q"].view(B, T, H, D)
    step = max(1, (1 << 27) // S)
    for b in range(B):
        n = lens[b]
        j = torch.arange(n, device="cuda")
        for h in range(H):
            if h % G == 0:
                if c.get("q4", True):
                    kk = _exact_rows(s["cache"][0][b, h // G, :n], s["cache"][1][b, h // G, :n], True, D)
                else:
                    kk = s["k_cache"][b, :n].view(n, Hk, D)[:, h // G].double()
                vv = _exact_rows(s["cache"][2][b, h // G, :n], s["cache"][3][b, h // G, :n], False, D) if c["op"] == "decode" else None
            for t in range(0, T, step):
                i = n - T + torch.arange(t, min(T, t + step), device="cuda")[:, None]
                x = q[b, t:t + step, h].double() @ kk.T * D ** -0.5
                x = x.masked_fill(~((j <= i) & ((j >= i - c["left"]) | (j < c["sinks"]))), -math.inf)
                if c["op"] == "decode":
                    lse[b, h, t:t + step] = torch.logsumexp(x, -1)
                    o[b, t:t + step, h] = torch.softmax(x, -1).nan_to_num(nan=0.0) @ vv
                else:
                    weights[b, h // G, :n] += torch.exp(x - s["lse"][b, h, t:t + step, None].double()).sum(0)
    return weights if c["op"] == "weigh" else {"o": o.flatten(-2), "lse": lse}
