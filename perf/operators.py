"""The operators around the sparse attention that are timed here, one dict per case.

``prep`` is the preparation of queries and keys (norm of each head, position
rotation) with its backward, ``append`` the same for new tokens of a serving
batch with their K/V rows written into the caches, ``window`` the attention with
a sliding window and sinks (forward, or a training step), ``wdecode`` its form for
new tokens over K/V caches and ``prefix`` the attention of a batch whose requests
share a long prefix.  ``own`` selects the package's kernels; without it the same
is computed by elementary torch operations in 32 bits.

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
BLOCK = 256  # queries per block of the plain banded attention


def _prep(B, N, H, Hk, D, dtype, R, interleaved=False, packed=False):
    return {"op": "prep", "B": B, "N": N, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "R": R,
            "interleaved": interleaved, "packed": packed}


def _append(B, T, H, Hk, D, dtype, S, R, interleaved=False):
    return {"op": "append", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "S": S, "R": R,
            "interleaved": interleaved}


def _window(B, N, H, Hk, D, dtype, left, right, sinks, train=True, ragged=False):
    return {"op": "window", "B": B, "N": N, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "left": left, "right": right,
            "sinks": sinks, "train": train, "ragged": ragged}


def _wdecode(B, T, H, Hk, D, dtype, S, left, sinks):
    return {"op": "wdecode", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "S": S, "left": left,
            "sinks": sinks}


def _prefix(B, T, H, Hk, D, dtype, P, S):
    return {"op": "prefix", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "dtype": dtype, "P": P, "S": S}


def listed():
    return [
        # One training layer's queries and keys at the benchmark's length, grouped K/V heads.
        {"name": "prep_32k", **_prep(1, 32768, 32, 8, 128, "bf16", 128)},
        # Packed sequences of odd lengths (positions given), part of the head rotated, neighbouring pairs, D = 80.
        {"name": "prep_ragged", **_prep(3, 1777, 12, 4, 80, "fp16", 32, interleaved=True, packed=True)},
        # The smallest call: one new token of one request.
        {"name": "append_1", **_append(1, 1, 8, 8, 64, "fp16", 4096, 64)},
        # One step of a large serving batch.
        {"name": "append_128", **_append(128, 1, 32, 8, 128, "bf16", 1024, 128)},
        # The small training step of the backward tables, causal, 256-token window: latency of a few workgroups.
        {"name": "window_2k", **_window(1, 2048, 8, 8, 128, "bf16", 255, 0, 4)},
        # The largest training layer: 32K tokens, 32 heads on 8, 1024-token window.
        {"name": "window_32k", **_window(1, 32768, 32, 8, 128, "bf16", 1023, 0, 4)},
        # A padded batch of ragged sequences, window to both sides, grouped heads of 64.
        {"name": "window_ragged", **_window(2, 10000, 12, 4, 64, "fp16", 300, 300, 16, ragged=True)},
        # Prompt processing with wide heads, eight query heads on each K/V head, forward only.
        {"name": "window_d256", **_window(2, 4096, 16, 2, 256, "bf16", 511, 0, 4, train=False)},
        # One request's next token over a 4096-token window: too few rows to fill the card.
        {"name": "wdecode_1", **_wdecode(1, 1, 32, 8, 128, "bf16", 8192, 4095, 4)},
        # The next tokens of a large batch of ragged requests.
        {"name": "wdecode_128", **_wdecode(128, 1, 32, 8, 128, "bf16", 8192, 4095, 4)},
        # A few requests behind a short system prompt, two tokens each (one drafted).
        {"name": "prefix_8", **_prefix(8, 2, 16, 4, 64, "fp16", 2048, 512)},
        # A large batch behind a long shared document.
        {"name": "prefix_64", **_prefix(64, 1, 32, 8, 128, "bf16", 32768, 1024)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes over the listed cases' ranges, odd ones among them, none dearer than the largest listed case of its kind."""
    while True:
        op = rng.choice(["prep", "append", "window", "window", "wdecode", "prefix"])
        dtype = rng.choice(["bf16", "fp16"])
        D = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        H = rng.choice([2, 4, 8, 12, 16, 32])
        Hk = H // rng.choice([g for g in (1, 2, 3, 4, 8) if H % g == 0])
        R = rng.choice([D, D, 32])
        inter = rng.random() < 0.4
        B = _log(rng, 1, 128)
        T = rng.choice([1, 1, 1, 2, 3, 5])
        if op == "prep":
            c = _prep(min(B, 4), _log(rng, 1, 32768), H, Hk, D, dtype, R, inter, rng.random() < 0.5)
            if c["B"] * c["N"] * (H + Hk) * D > 32768 * 40 * 128:
                continue
        elif op == "append":
            c = _append(B, T, H, Hk, D, dtype, _log(rng, 16, 4096), R, inter)
            if c["S"] < T or B * c["S"] * Hk * D > 128 * 1024 * 8 * 128:
                continue
        elif op == "window":
            left = _log(rng, 16, 4096) - 1
            right = rng.choice([0, 0, left, left // 3])
            c = _window(min(B, 4), _log(rng, 16, 32768), H, Hk, D, dtype, left, right, rng.choice([0, 1, 4, 16, 100]),
                        rng.random() < 0.7, rng.random() < 0.4)
            span = min(c["N"], left + right + 1 + BLOCK)
            if c["B"] * c["N"] * H * D * (span + c["sinks"]) > 32768 * 32 * 128 * (1024 + BLOCK + 4):
                continue
        elif op == "wdecode":
            c = _wdecode(B, T, H, Hk, D, dtype, _log(rng, 16, 16384), _log(rng, 16, 8192) - 1, rng.choice([0, 1, 4, 16, 100]))
            if c["S"] < T or B * c["S"] * Hk * D > 128 * 8192 * 8 * 128 or B * min(c["S"], c["left"] + 105) * Hk * D > 128 * 4100 * 8 * 128:
                continue
        else:
            c = _prefix(B, T, H, Hk, D, dtype, _log(rng, 64, 32768), _log(rng, 8, 2048))
            if c["S"] < T or B * T * H * D * c["P"] > 64 * 32 * 128 * 32768 or B * c["S"] * Hk * D > 64 * 1024 * 8 * 128:
                continue
        return c


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


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]

    def x(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dt)

    s = {"case": c}
    if c["op"] in ("prep", "append"):
        s["qw"], s["kw"] = (1 + 0.1 * torch.randn(D, generator=gen, device="cuda") for _ in range(2))
        s["cos"], s["sin"] = _tables(c["N"] if c["op"] == "prep" else c["S"], c["R"])
    if c["op"] == "prep":
        N = c["N"]
        s["q"], s["k"], s["dq"], s["dk"] = x(B, N, H * D), x(B, N, Hk * D), x(B, N, H * D), x(B, N, Hk * D)
        s["positions"] = None
        if c["packed"]:  # two sequences packed into each row, the cut anywhere
            cut = (torch.rand(B, 1, generator=gen, device="cuda") * N).int()
            at = torch.arange(N, device="cuda", dtype=torch.int32).expand(B, N)
            s["positions"] = torch.where(at >= cut, at - cut, at)
    elif c["op"] == "window":
        N = c["N"]
        s["q"], s["k"], s["v"] = x(B, N, H * D), x(B, N, Hk * D), x(B, N, Hk * D)
        s["do"] = x(B, N, H * D) if c["train"] else None
        s["lens"] = _lens(gen, B, N, 1) if c["ragged"] else None
    else:
        T, S = c["T"], c["S"]
        s["q"] = x(B, T, H * D)
        if c["op"] == "append":
            s["k"], s["v"] = x(B, T, Hk * D), x(B, T, Hk * D)
        s["k_cache"], s["v_cache"] = x(B, S, Hk * D), x(B, S, Hk * D)
        s["lens"] = _lens(gen, B, S, T)
        if c["op"] == "prefix":
            s["k_prefix"], s["v_prefix"] = x(c["P"], Hk * D), x(c["P"], Hk * D)
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
    H, Hk = c["H"], c["Hk"]
    if c["op"] == "prep":
        q, k, qw, kw = (s[n].detach().requires_grad_(True) for n in ("q", "k", "qw", "kw"))
        qo, ko = fta.flash_qk_norm_rope(q, k, H, s["cos"], s["sin"], qw, kw, eps=EPS, num_kv_heads=Hk,
                                        positions=s["positions"], interleaved=c["interleaved"])
        dq, dk, dqw, dkw = torch.autograd.grad((qo, ko), (q, k, qw, kw), (s["dq"], s["dk"]))
        return {"q": qo.detach(), "k": ko.detach(), "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}
    if c["op"] == "append":
        q = fta.flash_qk_norm_rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lens"], H, s["cos"],
                                          s["sin"], s["qw"], s["kw"], eps=EPS, num_kv_heads=Hk,
                                          interleaved=c["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if c["op"] == "window":
        win = (c["left"], c["right"])
        if not c["train"]:
            o, lse = fta.flash_window_attn(s["q"], s["k"], s["v"], H, win, c["sinks"], num_kv_heads=Hk,
                                           seq_lens=s["lens"])
            return {"o": o, "lse": lse}
        q, k, v = (s[n].detach().requires_grad_(True) for n in ("q", "k", "v"))
        o, lse = fta.flash_window_attn(q, k, v, H, win, c["sinks"], num_kv_heads=Hk, seq_lens=s["lens"])
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
        return {"o": o.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "wdecode":
        o, lse = fta.flash_window_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["lens"], H, c["left"], c["sinks"],
                                              num_kv_heads=Hk)
    else:
        o, lse = fta.flash_prefix_attn_decode(s["q"], s["k_prefix"], s["v_prefix"], s["k_cache"], s["v_cache"],
                                              s["lens"], H, num_kv_heads=Hk)
    return {"o": o, "lse": lse}


# ---------------------------------------------------------------- the plain forms


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] columns of x turned pair by pair."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, x[..., R:]), -1)


def _norm_rope(x, heads, w, cos, sin, interleaved):
    """(turned x, normed x without weight, reciprocal norm), heads split."""
    x = x.float().unflatten(-1, (heads, -1))
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n = x * r
    return _rotate(n * w, cos, sin, interleaved), n, r


def _norm_rope_back(dy, n, r, w, cos, sin, interleaved):
    g = _rotate(dy.float().unflatten(-1, n.shape[-2:]), cos, -sin, interleaved)
    h = g * w
    return (r * (h - n * (h * n).mean(-1, keepdim=True))).flatten(-2), (g * n).sum((0, 1, 2))


def _plain_prep(s, c):
    at = torch.arange(c["N"], device="cuda")[None] if s["positions"] is None else s["positions"].long()
    t = (s["cos"][at][:, :, None], s["sin"][at][:, :, None], c["interleaved"])
    qo, qn, qr = _norm_rope(s["q"], c["H"], s["qw"], *t)
    ko, kn, kr = _norm_rope(s["k"], c["Hk"], s["kw"], *t)
    dq, dqw = _norm_rope_back(s["dq"], qn, qr, s["qw"], *t)
    dk, dkw = _norm_rope_back(s["dk"], kn, kr, s["kw"], *t)
    dt = s["q"].dtype
    return {"q": qo.flatten(-2).to(dt), "k": ko.flatten(-2).to(dt), "dq": dq.to(dt), "dk": dk.to(dt), "dqw": dqw,
            "dkw": dkw}


def _plain_append(s, c):
    T = c["T"]
    at = s["lens"].long()[:, None] - T + torch.arange(T, device="cuda")
    t = (s["cos"][at][:, :, None], s["sin"][at][:, :, None], c["interleaved"])
    qo, ko = _norm_rope(s["q"], c["H"], s["qw"], *t)[0], _norm_rope(s["k"], c["Hk"], s["kw"], *t)[0]
    row = torch.arange(c["B"], device="cuda")[:, None]
    s["k_cache"][row, at] = ko.flatten(-2).to(s["k_cache"].dtype)
    s["v_cache"][row, at] = s["v"]
    return {"q": qo.flatten(-2).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _softmax(x, dim=-1):
    """(exp(x - max), its sum, log of the sum of exp(x)); a row of -inf gives zeros, zero and -inf."""
    m = x.amax(dim, keepdim=True)
    e = torch.exp(x - m.masked_fill(m == -math.inf, 0.0))
    l = e.sum(dim, keepdim=True)
    return e, l, (m + torch.log(l)).squeeze(dim)


def _plain_window(s, c):
    """Blocks of queries against the band of keys that they can see (and the sinks in front of it)."""
    B, N, H, Hk, D = c["B"], c["N"], c["H"], c["Hk"], c["D"]
    left, right, sinks = c["left"], c["right"], min(c["sinks"], N)
    G, w, scale, dt = H // Hk, min(BLOCK, N), D ** -0.5, s["q"].dtype
    nb = -(-N // w)
    rows = torch.arange(nb * w, device="cuda").view(nb, w)
    if w + left + right >= N:
        cols = torch.arange(N, device="cuda").expand(nb, N)
        real = torch.ones_like(cols, dtype=torch.bool)
    else:
        band = rows[:, :1] - left + torch.arange(w + left + right, device="cuda")
        first = torch.arange(sinks, device="cuda").expand(nb, sinks)
        cols = torch.cat((first, band), 1)
        real = torch.cat((first < band[:, :1], (band >= 0) & (band < N)), 1)  # each key once
    lens = torch.full((B,), N, device="cuda") if s["lens"] is None else s["lens"].long()
    i, j = rows[:, :, None], cols[:, None, :]
    seen = real[:, None] & (j <= i + right) & ((j >= i - left) | (j < sinks))
    seen = seen & (torch.maximum(i, j) < lens[:, None, None, None])  # [B, nb, w, cols]
    seen = seen[:, None, :, None].expand(B, 1, nb, G, w, cols.shape[1]).reshape(B, 1, nb, G * w, -1)
    at = cols.clamp(0, N - 1)

    def heads(x):  # [B, N, Hk * G * D] -> [B, Hk, nb, G * w, D]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, nb * w - N)).view(B, nb, w, Hk, -1, D)
        return x.permute(0, 3, 1, 4, 2, 5).reshape(B, Hk, nb, -1, D)

    def back(x):  # and back
        return x.view(B, Hk, nb, -1, w, D).permute(0, 2, 4, 1, 3, 5).reshape(B, nb * w, -1)[:, :N]

    def keys(x):
        return x.float().view(B, N, Hk, D).transpose(1, 2)[:, :, at]

    def to_keys(x):
        y = torch.zeros(B, Hk, N, D, device="cuda").index_add_(2, at.flatten(), x.flatten(2, 3))
        return y.transpose(1, 2).reshape(B, N, Hk * D).to(dt)

    q, k, v = heads(s["q"]), keys(s["k"]), keys(s["v"])
    p, l, lse = _softmax((q @ k.mT * scale).masked_fill_(~seen, -math.inf))
    p = p / l.clamp(min=1e-30)
    o = p @ v
    lse = lse.view(B, Hk, nb, G, w).permute(0, 1, 3, 2, 4).reshape(B, H, nb * w)[:, :, :N].contiguous()
    out = {"o": back(o).to(dt), "lse": lse}
    if c["train"]:
        do = heads(s["do"])
        ds = (do @ v.mT - (do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out |= {"dq": back(ds @ k).to(dt), "dk": to_keys(ds.mT @ q), "dv": to_keys(p.mT @ do)}
    return out


def _split_rows(x, Hk, D):
    """[B, T, H * D] -> [B, Hk, T * G, D]"""
    B, T = x.shape[:2]
    return x.float().view(B, T, Hk, -1, D).transpose(1, 2).reshape(B, Hk, -1, D)


def _join_rows(o, lse, c, dt):
    B, T, H, Hk, D = c["B"], c["T"], c["H"], c["Hk"], c["D"]
    o = o.view(B, Hk, T, H // Hk, D).transpose(1, 2).reshape(B, T, H * D)
    return {"o": o.to(dt), "lse": lse.view(B, Hk, T, H // Hk).transpose(2, 3).reshape(B, H, T)}


def _plain_wdecode(s, c):
    B, T, S, Hk, D, left = c["B"], c["T"], c["S"], c["Hk"], c["D"], c["left"]
    sinks, lens = min(c["sinks"], S), s["lens"].long()[:, None]
    if left + T + sinks >= S:
        cols = torch.arange(S, device="cuda").expand(B, S)
        real = torch.ones_like(cols, dtype=torch.bool)
    else:
        band = lens - T - left + torch.arange(left + T, device="cuda")
        first = torch.arange(sinks, device="cuda").expand(B, sinks)
        cols = torch.cat((first, band), 1)
        real = torch.cat((first < band[:, :1], band >= 0), 1)
    pos = (lens - T + torch.arange(T, device="cuda"))[:, :, None]
    j = cols[:, None]
    seen = real[:, None] & (j <= pos) & ((j >= pos - left) | (j < sinks))
    seen = seen.repeat_interleave(c["H"] // Hk, 1)[:, None]
    at, row = cols.clamp(0, S - 1), torch.arange(B, device="cuda")[:, None]
    k = s["k_cache"].view(B, S, Hk, D)[row, at].float().transpose(1, 2)
    v = s["v_cache"].view(B, S, Hk, D)[row, at].float().transpose(1, 2)
    x = (_split_rows(s["q"], Hk, D) @ k.mT * D ** -0.5).masked_fill(~seen, -math.inf)
    p, l, lse = _softmax(x)
    return _join_rows(p @ v / l.clamp(min=1e-30), lse, c, s["q"].dtype)


def _plain_prefix(s, c):
    B, T, S, P, Hk, D = c["B"], c["T"], c["S"], c["P"], c["Hk"], c["D"]
    q = _split_rows(s["q"], Hk, D) * D ** -0.5
    k1, v1 = (s[n].float().view(P, Hk, D).transpose(0, 1) for n in ("k_prefix", "v_prefix"))
    k2, v2 = (s[n].float().view(B, S, Hk, D).transpose(1, 2) for n in ("k_cache", "v_cache"))
    pos = s["lens"].long()[:, None] - T + torch.arange(T, device="cuda")
    seen = (torch.arange(S, device="cuda") <= pos[:, :, None]).repeat_interleave(c["H"] // Hk, 1)[:, None]
    flat = q.transpose(0, 1).reshape(Hk, -1, D)  # every request's rows against the one prefix
    x1 = (flat @ k1.mT).view(Hk, B, -1, P).transpose(0, 1)
    x2 = (q @ k2.mT).masked_fill(~seen, -math.inf)
    p, l, lse = _softmax(torch.cat((x1, x2), -1))
    o1 = (p[..., :P].transpose(0, 1).reshape(Hk, -1, P) @ v1).view(Hk, B, -1, D).transpose(0, 1)
    return _join_rows((o1 + p[..., P:] @ v2) / l, lse, c, s["q"].dtype)


PLAIN = {"prep": _plain_prep, "append": _plain_append, "window": _plain_window, "wdecode": _plain_wdecode,
         "prefix": _plain_prefix}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return PLAIN[state["case"]["op"]](state, state["case"])


# ---------------------------------------------------------------- work


def _pairs(N, left, right, sinks):
    """Visible (query, key) pairs of one sequence and head."""
    band = sum(min(N - 1, i + right) - max(0, i - left) + 1 for i in range(N))
    return band + sum(max(0, min(sinks, i - left, N)) for i in range(N))


def work(case):
    c = case
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    if c["op"] == "prep":
        n = B * c["N"] * (H + Hk) * D
        return {"bytes": 8 * n + 4 * c["N"] * c["R"] + 16 * D, "flops": 20 * n}
    if c["op"] == "append":
        n = B * c["T"]
        return {"bytes": 4 * n * (H + 2 * Hk) * D + 4 * n * c["R"], "flops": 8 * n * (H + Hk) * D}
    if c["op"] == "window":
        N = c["N"]
        pairs = B * H * _pairs(N, c["left"], c["right"], min(c["sinks"], N))
        if c["ragged"]:  # lengths of half to all of N
            pairs = int(pairs * (1 if B == 1 else (1 + 0.75 * (B - 1)) / B))
        nbytes = 4 * B * N * (H + Hk) * D + 4 * B * H * N
        if c["train"]:
            nbytes += 4 * B * N * (H + Hk) * D
        return {"bytes": nbytes, "flops": (14 if c["train"] else 4) * D * pairs}
    T, S = c["T"], c["S"]
    rows = B * T * H
    tokens = S if B == 1 else S * (1 + 0.75 * (B - 1)) / B  # the mean length
    if c["op"] == "wdecode":
        seen = int(B * min(tokens, c["left"] + T + c["sinks"]))
        shared = 0
    else:
        seen, shared = int(B * tokens), c["P"]
    return {"bytes": 4 * (seen + shared) * Hk * D + 4 * rows * D + 4 * rows,
            "flops": 4 * D * (H * T * seen + rows * shared)}


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
    return torch.cat((z, rest), -1).flatten(-2)


def _exact_rows(q, k, v, seen, do=None):
    """One head in float64: q [n, D], k, v [m, D], seen [n, m]; (o, lse) and the gradients of q, k, v."""
    x = (q @ k.T * q.shape[-1] ** -0.5).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
    o = p @ v
    if do is None:
        return o, lse
    ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) * q.shape[-1] ** -0.5
    return o, lse, ds @ k, ds.T @ q, p.T @ do


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    G = H // Hk
    if c["op"] == "prep":
        pos = torch.arange(c["N"], device="cuda").expand(B, -1) if s["positions"] is None else s["positions"]
        ins = [s[n].double().requires_grad_(True) for n in ("q", "k", "qw", "kw")]
        outs = (_exact_turned(ins[0], H, ins[2], c, pos), _exact_turned(ins[1], Hk, ins[3], c, pos))
        grads = torch.autograd.grad(outs, ins, (s["dq"].double(), s["dk"].double()))
        return dict(zip(("q", "k", "dq", "dk", "dqw", "dkw"), (*(x.detach() for x in outs), *grads)))
    if c["op"] == "append":
        T = c["T"]
        found = {"q": torch.zeros(B, T, H * D, device="cuda", dtype=torch.float64), "k_cache": s["k_cache"].double(),
                 "v_cache": s["v_cache"].double()}
        first = s["lens"].long() - T
        pos = first[:, None] + torch.arange(T, device="cuda")
        found["q"] = _exact_turned(s["q"].double(), H, s["qw"].double(), c, pos)
        new = _exact_turned(s["k"].double(), Hk, s["kw"].double(), c, pos)
        for b, f in enumerate(first.tolist()):
            found["k_cache"][b, f:f + T], found["v_cache"][b, f:f + T] = new[b], s["v"][b].double()
        return found
    f64 = dict(device="cuda", dtype=torch.float64)
    N = c["N"] if c["op"] == "window" else c["T"]
    out = {"o": torch.zeros(B, N, H, D, **f64), "lse": torch.full((B, H, N), -math.inf, **f64)}
    train = c["op"] == "window" and c["train"]
    if train:
        out |= {"dq": torch.zeros(B, N, H, D, **f64), "dk": torch.zeros(B, N, Hk, D, **f64),
                "dv": torch.zeros(B, N, Hk, D, **f64)}
    lens = None if s["lens"] is None else s["lens"].tolist()
    for b in range(B):
        if c["op"] == "window":
            n = m = N if lens is None else lens[b]
            kk, vv = (s[x][b].view(N, Hk, D) for x in ("k", "v"))
            i, left, right = torch.arange(n, device="cuda"), c["left"], c["right"]
        else:
            n, m = c["T"], lens[b]
            kk, vv = (s[x][b].view(-1, Hk, D) for x in ("k_cache", "v_cache"))
            i, left, right = m - n + torch.arange(n, device="cuda"), c.get("left", m), 0
        sinks, step = c.get("sinks", 0), 1024
        for r in range(0, n, step):
            ir = i[r:r + step, None]
            j = torch.arange(m, device="cuda")
            seen = (j <= ir + right) & ((j >= ir - left) | (j < sinks))
            j = seen.any(0).nonzero()[:, 0]
            seen = seen[:, j]
            for h in range(H):
                kj, vj = kk[j, h // G].double(), vv[j, h // G].double()
                see = seen
                if c["op"] == "prefix":
                    kp, vp = (s[x].view(-1, Hk, D)[:, h // G].double() for x in ("k_prefix", "v_prefix"))
                    kj, vj = torch.cat((kp, kj)), torch.cat((vp, vj))
                    see = torch.cat((torch.ones(seen.shape[0], kp.shape[0], device="cuda", dtype=torch.bool), seen), 1)
                at = (b, slice(r, min(n, r + step)), h)
                q = s["q"][b].view(N, H, D)[at[1], h].double()
                do = s["do"][b].view(N, H, D)[at[1], h].double() if train else None
                got = _exact_rows(q, kj, vj, see, do)
                out["o"][at], out["lse"][b, h, at[1]] = got[0], got[1]
                if train:
                    out["dq"][at] = got[2]
                    out["dk"][b].index_put_((j, torch.tensor(h // G, device="cuda")), got[3], accumulate=True)
                    out["dv"][b].index_put_((j, torch.tensor(h // G, device="cuda")), got[4], accumulate=True)
    return {n: x if n == "lse" else x.flatten(-2) for n, x in out.items()}
