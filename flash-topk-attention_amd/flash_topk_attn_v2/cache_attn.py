"""Attention of new tokens over K/V caches (HIP, gfx950): the launch that the window and
the shared-prefix forms have in common, and the shared-prefix form.

No counterpart in the reference.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import _lib
from .qk_prep import check_cache


@lru_cache(maxsize=1024)
def _geometry(what, q, dtype, num_heads, num_kv_heads, S, P, left, sinks, scale):
    """``(H, Hk, D, left, scale, workspace bytes)``, checked (calls of one shape are checked once)."""
    if len(q) != 3:
        raise ValueError(f"{what}: q must be [B, T, num_heads * D]")
    if dtype not in _lib.HALVES:
        raise ValueError(f"{what}: q must be float16 or bfloat16")
    B, T, C = q
    H, Hk, D = _lib.head_counts(what, C, num_heads, num_kv_heads)
    if B == 0 or T == 0:
        raise ValueError(f"{what}: empty batch or no new tokens")
    _lib.int_sizes(what, B, T, S, P)
    left = S if left is None else left
    nbytes = int(_lib.lib().fta_cache_attn_workspace_size(B, H, Hk, T, S, D, P, left, sinks))
    return H, Hk, D, left, _lib.softmax_scale(what, scale, D), nbytes


def cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, k_prefix, v_prefix, left, sinks, scale):
    """Checks and the launch of ``fta_cache_attn``."""
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _lib.no_grad_inputs(what, q, k_cache, v_cache, k_prefix, v_prefix)
    S = k_cache.shape[1] if k_cache.ndim == 3 else 0
    P = 0 if k_prefix is None else k_prefix.shape[0]
    num_heads, num_kv_heads, scale = _lib.scalars(what, num_heads, num_kv_heads, scale)
    H, Hk, D, left, scale, nbytes = _geometry(what, q.shape, q.dtype, num_heads, num_kv_heads, S, P, left, sinks, scale)
    B, T, _ = q.shape
    check_cache(what, q, k_cache, v_cache, cache_lens, B, Hk * D)
    kpa = kps = vpa = vps = None
    if k_prefix is not None:
        if k_prefix.ndim != 2 or k_prefix.shape[1] != Hk * D or v_prefix.shape != k_prefix.shape:
            raise ValueError(f"{what}: k_prefix and v_prefix must be [P, num_kv_heads * D] = [P, {Hk * D}]")
        if k_prefix.dtype != q.dtype or v_prefix.dtype != q.dtype:
            raise ValueError(f"{what}: the prefix must have q's type")
        _lib.check_device(what, q.device, k_prefix, v_prefix)
        if P > 0:
            kpa, kps = _lib.rows_in_place(what, k_prefix[None], Hk)
            vpa, vps = _lib.rows_in_place(what, v_prefix[None], Hk)
    kca, kcs = _lib.rows_in_place(what, k_cache, Hk)
    vca, vcs = _lib.rows_in_place(what, v_cache, Hk)
    q, qa, qs = _lib.rows(q, H)
    lens = cache_lens.contiguous()
    dev = q.device
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(B, H, T, device=dev, dtype=torch.float32)
    ws = _lib.workspace(nbytes, dev) if nbytes else None
    _lib.call("fta_cache_attn", dev, qa, qs, kca, kcs, vca, vcs, _lib.DTYPE_CODES[q.dtype], B, H, Hk, T, S, D,
              lens.data_ptr(), kpa, kps, vpa, vps, P, left, sinks, scale, o.data_ptr(), _lib.dense_strides(q.shape, H),
              lse.data_ptr(), _lib.ptr(ws), nbytes)
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
    nothing gives o = 0, lse = -inf.  Cache rows that no token sees may hold anything.
    Probabilities are rounded to the inputs' type, as in ``flash_window_attn``.  Not
    differentiable.

    Returns ``(output [B, T, num_heads * D], lse [B, num_heads, T] float32)``.
    """
    what = "flash_prefix_attn_decode"
    if k_prefix is None or v_prefix is None:
        raise ValueError(f"{what}: k_prefix and v_prefix are required")
    return cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, k_prefix, v_prefix, None, 0, scale)


__all__ = ["flash_prefix_attn_decode"]
