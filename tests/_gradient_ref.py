"""Gradients of the window attention in float64 with delta formed from a given 16-bit output, as the
kernels form it from their own, and what they may be off by (test infrastructure).

``_operators_ref.attend`` takes delta from the exact output and allows for its rounding in every dS at
its worst, which for dK is most of the bound.  From the output itself delta is exact but for
an fp32 sum of D products (within F of its terms), and the bound is that of the rounded dS.
"""

import math

import torch

import _operators_ref as R


def head(q, k, v, seen, scale, dtype, do, o16, delta_factor=1.0):
    """One head (2-D float64 tensors): dq, dk and their elementwise bounds.  ``delta_factor``: a planted mistake."""
    u, t = R.half_step(dtype), R.tiny(dtype)
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[:, None]).masked_fill(~seen, 0.0)
    dp = do @ v.T
    delta = (do * o16).sum(-1, keepdim=True)
    ds = p * (dp - delta_factor * delta)
    terms = do.abs() @ v.abs().T + (do * o16).abs().sum(-1, keepdim=True)
    ds_off = p * R.F * terms + 2 * R.F * ds.abs() + R.FLUSH * terms * seen.double()
    off = ds_off + u * (ds.abs() + ds_off) + (t + R.FLUSH) * seen.double()
    return {"dq": scale * (ds @ k), "dk": scale * (ds.T @ q),
            "dq_tol": u * scale * (ds @ k).abs() + scale * (off + R.F * ds.abs()) @ k.abs() * (1 + u) + t,
            "dk_tol": scale * (off + R.F * ds.abs()).T @ q.abs() * (1 + u)}


def window(q, k, v, o, do, H, Hk, left, right, sinks, scale, lens=None, delta_factor=1.0):
    """dq and dk of ``flash_window_attn`` whose output was ``o``, with bounds; padding rows are zero."""
    B, N, C = q.shape
    D, G, dtype, dev = C // H, H // Hk, q.dtype, q.device
    out = {n: torch.zeros(B, N, heads, D, device=dev, dtype=torch.float64)
           for n, heads in (("dq", H), ("dq_tol", H), ("dk", Hk), ("dk_tol", Hk))}
    for b in range(B):
        n = N if lens is None else max(0, min(N, int(lens[b])))
        if n == 0:
            continue
        seen = R.window_mask(n, n, 0, left, right, sinks, dev)
        for h in range(H):
            at = lambda x, i, heads: x[b, :n].view(n, heads, D)[:, i].double()  # noqa: E731
            r = head(at(q, h, H), at(k, h // G, Hk), at(v, h // G, Hk), seen, scale, dtype, at(do, h, H), at(o, h, H),
                     delta_factor)
            out["dq"][b, :n, h], out["dq_tol"][b, :n, h] = r["dq"], r["dq_tol"]
            out["dk"][b, :n, h // G] += r["dk"]
            out["dk_tol"][b, :n, h // G] += r["dk_tol"]
    out["dk_tol"] += R.half_step(dtype) * out["dk"].abs() + R.tiny(dtype)
    return {n: x.flatten(-2) for n, x in out.items()}


# dtype, B, N, H, Hk, D, left, right, sinks, lens
CASES = [
    (torch.bfloat16, 1, 90, 2, 1, 64, 20, 4, 3, None),
    (torch.bfloat16, 1, 130, 4, 2, 128, 40, 0, 4, None),
    (torch.float16, 2, 130, 3, 1, 48, 63, 31, 0, [130, 70]),
    (torch.bfloat16, 1, 60, 2, 1, 80, 2, 0, 1, None),
    (torch.bfloat16, 1, 100, 2, 2, 96, 30, 0, 2, None),
    (torch.float16, 1, 200, 4, 1, 128, 200, 0, 0, None),
    (torch.bfloat16, 2, 140, 2, 1, 256, 50, 9, 5, [140, 33]),
    (torch.float16, 1, 110, 2, 2, 160, 25, 25, 40, None),
]


def inputs(case, device, seed=7):
    """q, k, v, do of a case."""
    from _helpers import rand

    dtype, B, N, H, Hk, D = case[:6]
    q, do = (rand((B, N, H * D), seed + i, dtype, device) for i in (0, 1))
    k, v = (rand((B, N, Hk * D), seed + i, dtype, device) for i in (2, 3))
    return q, k, v, do


def slope_along(case, q, k, v, do, name, direction, h=1e-5):
    """Change of sum(o do) in float64 over a central step of +- h along ``direction`` of q, k or v."""
    _, B, N, H, Hk, D, left, right, sinks, lens = case

    def loss(step):
        x = {"dq": q, "dk": k, "dv": v}
        x = {n: t.double() + (step * direction if n == name else 0.0) for n, t in x.items()}
        total = 0.0
        for b in range(B):
            n = N if lens is None else lens[b]
            seen = R.window_mask(n, n, 0, left, right, sinks, q.device)
            for i in range(H):
                a, c, d = (x[m][b, :n].view(n, heads, D)[:, j] for m, heads, j in
                           (("dq", H, i), ("dk", Hk, i * Hk // H), ("dv", Hk, i * Hk // H)))
                p = torch.softmax((a @ c.T * D ** -0.5).masked_fill(~seen, -math.inf), -1)
                total = total + ((p @ d) * do[b, :n].view(n, H, D)[:, i].double()).sum()
        return total

    return float((loss(h) - loss(-h)) / (2 * h))


def along(case, q, k, v, do, ref, name):
    """(direction, slope along it, worst-case error of a gradient's sum along it): the direction is the
    gradient's own, so that the slope is the largest there is."""
    d = ref[name] / ref[name].square().mean().sqrt()
    return d, slope_along(case, q, k, v, do, name, d), float((ref[name + "_tol"] * d.abs()).sum())
