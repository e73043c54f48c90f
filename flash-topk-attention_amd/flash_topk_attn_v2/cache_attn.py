"""Attention of new tokens over K/V caches (HIP, gfx950): the launch that the window and
the shared-prefix forms have in common, and the shared-prefix form.

No counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .qk_prep import _cache_strides, _check_cache, _no_grad_inputs


def cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, k_prefix, v_prefix, left, sinks, scale):
    """Checks and the launch of ``fta_cache_attn``."""
    if q.ndim != 3:
        raise ValueError(f"{what}: q must be [B, T, num_heads * D]")
    if q.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what}: q must be float16 or bfloat16")
    _no_grad_inputs(what, q, k_cache, v_cache, k_prefix, v_prefix)
    B, T, C = q.shape
    H, Hk, D = _lib.head_counts(what, C, num_heads, num_kv_heads)
    if B == 0 or T == 0:
        raise ValueError(f"{what}: empty batch or no new tokens")
    _check_cache(what, k_cache, v_cache, cache_lens, B, Hk, D, q)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 3.0e38:
        raise ValueError(f"{what}: scale must be positive and finite")
    S, P, kps, vps = k_cache.shape[1], 0, None, None
    if left is None:
        left = S
    if k_prefix is not None:
        if k_prefix.ndim != 2 or k_prefix.shape[1] != Hk * D or v_prefix.shape != k_prefix.shape:
            raise ValueError(f"{what}: k_prefix and v_prefix must be [P, num_kv_heads * D] = [P, {Hk * D}]")
        if k_prefix.dtype != q.dtype or v_prefix.dtype != q.dtype:
            raise ValueError(f"{what}: the prefix must have q's type")
        _lib.check_tensors(what, q.device, k_prefix=k_prefix, v_prefix=v_prefix)
        P = k_prefix.shape[0]
        if P > 0:
            kps, vps = (_cache_strides(what, x[None], D) for x in (k_prefix, v_prefix))
    kcs, vcs = _cache_strides(what, k_cache, D), _cache_strides(what, v_cache, D)
    dev = q.device
    qq, qs = _lib.token_view(q, "bnc", H)
    lens = cache_lens.contiguous()
    o = torch.empty(B, T, C, device=dev, dtype=q.dtype)
    lse = torch.empty(B, H, T, device=dev, dtype=torch.float32)
    nbytes = _lib.size_of("fta_cache_attn_workspace_size", B, H, Hk, T, S, D, P, left, sinks)
    ws = _lib.workspace(nbytes, dev) if nbytes else None
    with _lib.on_device(dev):
        rc = _lib.lib().fta_cache_attn(
            _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(k_cache), kcs, _lib.ptr(v_cache), vcs, _lib.dtype_code(q.dtype),
            B, H, Hk, T, S, D, _lib.ptr(lens), _lib.ptr(k_prefix), kps, _lib.ptr(v_prefix), vps, P, left, sinks, scale,
            _lib.ptr(o), _lib.i64arr((T * C, D, C)), _lib.ptr(lse), _lib.ptr(ws), nbytes, _lib.stream_ptr(dev))
    _lib.check(rc, what)
    return o, lse


def flash_prefix_attn_decode(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_lens: torch.Tensor,
    num_heads: int,
    scale: Optional[float] = None,
    num_kv_heads: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of the last T tokens of each request, whose sequences all begin with one
    shared prefix: the prefix's K and V are read once for the whole batch.

    ``q`` is ``[B, T, num_heads * D]``, ``k_prefix`` and ``v_prefix`` ``[P, num_kv_heads *
    D]`` (P may be 0), the caches ``[B, S, num_kv_heads * D]`` hold what comes after the
    prefix.  ``cache_lens`` (int32 ``[B]`` on the device, not read by the host) counts each
    request's own tokens with these T; values outside ``[0, S]`` are clamped.  Token t sees
    the whole prefix and own key j when ``j <= cache_lens[b] - T + t``; one that sees
    nothing gives o = 0, lse = -inf.  Cache rows that no token sees may hold anything.  Not
    differentiable.

    Returns ``(output [B, T, num_heads * D], lse [B, num_heads, T] float32)``.
    """
    what = "flash_prefix_attn_decode"
    if k_prefix is None or v_prefix is None:
        raise ValueError(f"{what}: k_prefix and v_prefix are required")
    return cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, k_prefix, v_prefix, None, 0, scale)


__all__ = ["flash_prefix_attn_decode"]
