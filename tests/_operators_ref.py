"""Plain float64 forms of the operators around the sparse attention, and how far a result
in 16 bits may be from them (test infrastructure).

u is half a step of the type, relative.  What a kernel rounds, and so may be off by:
its outputs (u of the value), P and dS before the second product of each pair (u of
every term, and half a subnormal step where fp16 ends), and fp32 arithmetic.  The
latter is bounded by F = 3e-4 of the terms' magnitudes: with unit-variance inputs and D
up to 256 a score of D products summed in fp32 is off by at most D 2^-24 sum |q k| scale
< 256 * 6e-8 * 16 = 2.5e-4 in the exponent in the worst case, exp2 and the sums by a few
2^-23 more.  exp2 and bf16 end at 2^-126: a P below it is taken as 0, an absolute error of
at most FLUSH = 2^-126 in every P (and of FLUSH |dP - delta| in dS).
"""

import math

import torch

F = 3e-4
FLUSH = 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a subnormal step: the absolute rounding where the type's exponents end."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def window_mask(n, m, first, left, right, sinks, device):
    """[n, m]: which of m keys query ``first + i`` sees."""
    i = first + torch.arange(n, device=device)[:, None]
    j = torch.arange(m, device=device)
    return (j <= i + right) & ((j >= i - left) | (j < sinks)) & (i >= 0)


def attend(q, k, v, seen, scale, dtype, do=None, o16=None):
    """One head in float64 (2-D tensors): dict of values and of elementwise bounds.

    ``o16``: the 16-bit output that the backward forms delta from.
    """
    u, t = half_step(dtype), tiny(dtype)
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
    p = p.masked_fill(~seen, 0.0)
    o = p @ v
    seen64 = seen.double()
    mag = p @ v.abs()
    r = {"o": o, "lse": lse, "o_tol": u * o.abs() + (u + F) * mag + (t + FLUSH) * (1 + seen64 @ v.abs()),
         "lse_tol": F + 1e-6 * lse.abs().nan_to_num(posinf=0.0)}
    if do is None:
        return r
    dp = do @ v.T
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    d_off = (do.abs() * (r["o_tol"])).sum(-1, keepdim=True)  # delta comes from the rounded o
    terms = do.abs() @ v.abs().T + (do * o).abs().sum(-1, keepdim=True)  # of dP - delta
    ds_off = p * (F * terms + d_off) + 2 * F * ds.abs() + FLUSH * terms * seen64
    off = ds_off + u * (ds.abs() + ds_off) + (t + FLUSH) * seen64
    r |= {"dq": scale * (ds @ k), "dk": scale * (ds.T @ q), "dv": p.T @ do}
    r["dq_tol"] = u * r["dq"].abs() + scale * (off + F * ds.abs()) @ k.abs() * (1 + u) + t
    r["dk_tol"] = scale * (off + F * ds.abs()).T @ q.abs() * (1 + u)  # rounding of the output: once per shared head sum
    r["dv_tol"] = ((u + F) * p + (t + FLUSH) * seen64).T @ do.abs() * (1 + u)
    return r


def window(q, k, v, H, Hk, left, right, sinks, scale, lens=None, do=None):
    """``flash_window_attn`` in float64 with bounds, on q's device; padding rows are o = 0, lse = -inf."""
    B, N, C = q.shape
    D, G, dtype, dev = C // H, H // Hk, q.dtype, q.device
    f64 = dict(device=dev, dtype=torch.float64)
    out = {"o": torch.zeros(B, N, H, D, **f64), "lse": torch.full((B, H, N), -math.inf, **f64)}
    if do is not None:
        out |= {"dq": torch.zeros(B, N, H, D, **f64), "dk": torch.zeros(B, N, Hk, D, **f64),
                "dv": torch.zeros(B, N, Hk, D, **f64)}
    out |= {n + "_tol": torch.zeros_like(x) for n, x in list(out.items())}
    for b in range(B):
        n = N if lens is None else max(0, min(N, int(lens[b])))
        if n == 0:
            continue
        seen = window_mask(n, n, 0, left, right, sinks, dev)
        for h in range(H):
            at = lambda x, i, heads: x[b, :n].view(n, heads, D)[:, i].double()  # noqa: E731
            r = attend(at(q, h, H), at(k, h // G, Hk), at(v, h // G, Hk), seen, scale, dtype,
                       None if do is None else at(do, h, H))
            for name in ("o", "o_tol", "dq", "dq_tol"):
                if name in r:
                    out[name][b, :n, h] = r[name]
            for name in ("lse", "lse_tol"):
                out[name][b, h, :n] = r[name]
            if do is not None:
                for name in ("dk", "dk_tol", "dv", "dv_tol"):
                    out[name][b, :n, h // G] += r[name]
    if do is not None:
        for name in ("dk", "dv"):
            out[name + "_tol"] += half_step(dtype) * out[name].abs() + tiny(dtype)
    return {n: x if n.startswith("lse") else x.flatten(-2) for n, x in out.items()}


def cache(q, k_cache, v_cache, lens, H, Hk, left, sinks, scale, k_prefix=None, v_prefix=None):
    """``flash_window_attn_decode`` / ``flash_prefix_attn_decode`` in float64 with bounds."""
    B, T, C = q.shape
    D, G, S, dev = C // H, H // Hk, k_cache.shape[1], q.device
    out = {"o": torch.zeros(B, T, H, D, device=dev, dtype=torch.float64),
           "lse": torch.full((B, H, T), -math.inf, device=dev, dtype=torch.float64)}
    out |= {n + "_tol": torch.zeros_like(x) for n, x in list(out.items())}
    for b in range(B):
        n = max(0, min(S, int(lens[b])))
        seen = window_mask(T, n, n - T, left, 0, sinks, dev)
        for h in range(H):
            kk, vv = (x[b, :n].reshape(n, Hk, D)[:, h // G].double() for x in (k_cache, v_cache))
            see = seen
            if k_prefix is not None:
                kp, vp = (x.reshape(-1, Hk, D)[:, h // G].double() for x in (k_prefix, v_prefix))
                kk, vv = torch.cat((kp, kk)), torch.cat((vp, vv))
                see = torch.cat((torch.ones(T, kp.shape[0], device=dev, dtype=torch.bool), seen), 1)
            if kk.shape[0] == 0:
                continue
            r = attend(q[b].view(T, H, D)[:, h].double(), kk, vv, see, scale, q.dtype)
            dead = ~see.any(-1)
            for name in ("o", "o_tol"):
                out[name][b, :, h] = r[name].masked_fill(dead[:, None], 0.0)
            for name in ("lse", "lse_tol"):
                out[name][b, h] = r[name]
    return {n: x if n.startswith("lse") else x.flatten(-2) for n, x in out.items()}


def turned(x, heads, w, cos, sin, pos, eps, interleaved):
    """``flash_qk_norm_rope`` of one tensor in float64 (differentiable)."""
    B, N = x.shape[:2]
    x = x.view(B, N, heads, -1)
    u = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    u = u if w is None else u * w
    pos = pos.long().clamp(0, cos.shape[0] - 1)
    c, s = (t.double()[pos][:, :, None] for t in (cos, sin))
    R = 2 * cos.shape[1]
    if interleaved:
        a, b = u[..., 0:R:2], u[..., 1:R:2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = u[..., :R // 2], u[..., R // 2:R]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, u[..., R:]), -1).flatten(-2)


def check(got, ref, names, what=""):
    """Every element of every output within its bound; infinities and NaN in the same places."""
    for name in names:
        g, r, tol = got[name].detach().double(), ref[name], ref[name + "_tol"]
        assert g.shape == r.shape, f"{what} {name}: {tuple(g.shape)} instead of {tuple(r.shape)}"
        fine = r.isfinite()
        assert torch.equal(g[~fine], r[~fine]), f"{what} {name}: infinite values differ"
        assert g[fine].isfinite().all(), f"{what} {name}: values that are not finite"
        off = (g - r)[fine].abs()
        over = off > tol[fine]
        assert not over.any(), (f"{what} {name}: {int(over.sum())} of {over.numel()} elements off, worst "
                                f"{float((off / tol[fine].clamp(min=1e-300)).max()):.2f} times its bound")
