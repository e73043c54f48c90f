"""4-bit caches in float64, and how far results over them may be off (test infrastructure).

Codes and scales are integers and float16 numbers: what a cache holds is compared exactly.

Attention multiplies the codes as 16 + n and takes 24 times the sum of their partners off again.
Its score is a sum over groups of d (sum of q (16 + n) - 24 sum of q): a group's product adds 32
terms of up to 31 |q| to a first addend of 24 sum |q|, each addition off by at most 2^-24 of what
it has reached (below 55 sum |q|), 40 of them with those that form the first addend.  For unit-variance
q of D = 256 that is 40 * 2^-24 * 55 * sum |q| d scale < 40 * 6e-8 * 55 * 210 * 0.35 / 16 = 6.1e-4 in
the exponent, beside the 3e-4 of the other fp32 arithmetic: F4 = 1e-3.  The output's sums reach
55 sum p |d|, in two additions per 64 keys and two for their ones.
"""

import math

import torch

import _operators_ref as R

F4 = 1e-3


def quantize(x):
    """``(codes n [..., groups, 32], scales float16 [..., groups])`` of rows [..., D] of 16-bit values."""
    x = torch.nn.functional.pad(x.double(), (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    hi, lo = x.amax(-1), x.amin(-1)
    d = (torch.where(-lo >= hi, lo, hi) / -8).clamp(-65504, 65504).to(torch.float16)
    n = torch.where(d[..., None] == 0, 8.0, torch.round(x / d[..., None].double()) + 8).clamp(0, 15)
    return n.long(), d


def pack(n, key):
    """The bytes of codes [..., groups, 32]."""
    n = n.unflatten(-1, (4, 8))
    n = (n.transpose(-2, -3) if key else n).flatten(-3)
    return (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8)


def values(codes, scales, key, D):
    """What rows hold, float64 [..., D], and |d| of each column's group."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    g = scales.shape[-1]
    n = n.unflatten(-1, (4, g, 8)).transpose(-2, -3) if key else n.unflatten(-1, (g, 4, 8))
    d = scales.double()[..., None].expand(*scales.shape, 32)
    return ((n.flatten(-2) - 8) * d).flatten(-2)[..., :D], d.abs().flatten(-2)[..., :D]


def cache(B, S, Hk, D, device, seed, scale=1.0):
    """A full ``Q4Cache`` of normal values."""
    import flash_topk_attn_v2 as fta

    c = fta.flash_q4_cache(B, S, Hk, D, device)
    gen = torch.Generator().manual_seed(seed)
    for key, codes, scales in ((True, c.k_codes, c.k_scales), (False, c.v_codes, c.v_scales)):
        n, d = quantize((torch.randn(B, Hk, S, D, generator=gen) * scale).to(torch.bfloat16))
        codes.copy_(pack(n, key))
        scales.copy_(d)
    return c


def attend(q, c, lens, H, Hk, left, sinks, scale):
    """``flash_window_attn_decode_q4`` in float64 with bounds."""
    B, T, C = q.shape
    D, G, S, dev, dt = C // H, H // Hk, c.k_codes.shape[2], q.device, q.dtype
    u, t = R.half_step(dt), R.tiny(dt)
    # Of p d.  bf16 keeps 8 bits, 2^e (1 + m / 128): half a step is 2^(e - 8), at most 2^-8 of a value of 2^e and more.
    # Two of them, hi + lo: |lo| is at most 2^-8 |x|, and its own rounding 2^-8 of that, 2^-16 |x|.
    up = 2.0 ** -16 if dt == torch.float16 else 2.0 ** -8
    out = {"o": torch.zeros(B, T, H, D, device=dev, dtype=torch.float64),
           "lse": torch.full((B, H, T), -math.inf, device=dev, dtype=torch.float64)}
    out |= {n + "_tol": torch.zeros_like(x) for n, x in list(out.items())}
    for b in range(B):
        n = max(0, min(S, int(lens[b])))
        if n == 0:
            continue
        see = R.window_mask(T, n, n - T, left, 0, sinks, dev)
        dead = ~see.any(-1)
        for h in range(H):
            kk, _ = values(c.k_codes[b, h // G, :n], c.k_scales[b, h // G, :n], True, D)
            vv, d = values(c.v_codes[b, h // G, :n], c.v_scales[b, h // G, :n], False, D)
            s = (q[b].view(T, H, D)[:, h].double() @ kk.T * scale).masked_fill(~see, -math.inf)
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - lse.masked_fill(dead, 0.0)[:, None]).masked_fill(~see, 0.0)
            o = p @ vv
            adds = (4 * -(-n // 64) + 64) * 2.0 ** -24
            out["o"][b, :, h] = o
            out["o_tol"][b, :, h] = (u * o.abs() + (up + F4) * (p @ vv.abs()) + adds * 55 * (p @ d) + t + R.FLUSH * d.sum(0) * 8)
            out["lse"][b, h], out["lse_tol"][b, h] = lse, F4 + 1e-6 * lse.abs().nan_to_num(posinf=0.0)
    return {n: x if n.startswith("lse") else x.flatten(-2) for n, x in out.items()}
