"""Sliding-window attention with sinks (HIP, gfx950): the local layers beside the
top-k sparse ones, forward and backward, and its form for new tokens over K/V caches.

No counterpart in the reference.
"""

from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .cache_attn import cache_attn

_MAX = (1 << 30) - 1  # windows past this are the same as this


@lru_cache(maxsize=1024)
def _geometry(what, q, k, v, dtypes, num_heads, num_kv_heads, window, num_sinks, scale):
    """``(H, Hk, D, left, right, sinks, scale)``, checked (calls of one shape are checked once)."""
    if len(q) != 3 or len(k) != 3 or len(v) != 3:
        raise ValueError(f"{what}: q, k and v must be [B, N, heads * D]")
    if dtypes[0] not in _lib.HALVES or dtypes != (dtypes[0],) * 3:
        raise ValueError(f"{what}: q, k and v must all be float16 or all bfloat16")
    B, N, C = q
    H, Hk, D = _lib.head_counts(what, C, num_heads, num_kv_heads)
    if B == 0 or N == 0:
        raise ValueError(f"{what}: empty batch or sequence")
    if tuple(k) != (B, N, Hk * D) or tuple(v) != (B, N, Hk * D):
        raise ValueError(f"{what}: k and v must be [B, N, num_kv_heads * D] = {[B, N, Hk * D]}")
    _lib.int_sizes(what, B, N)
    if len(window) != 2 or min(window) < 0:
        raise ValueError(f"{what}: window must be (left, right), both non-negative")
    if num_sinks < 0:
        raise ValueError(f"{what}: num_sinks must be non-negative")
    left, right, sinks = (min(x, _MAX) for x in (*window, num_sinks))
    return H, Hk, D, left, right, sinks, _lib.softmax_scale(what, scale, D)


class _WindowAttnFunc(torch.autograd.Function):
    """Autograd function behind ``flash_window_attn``."""

    @staticmethod
    def forward(ctx, q, k, v, lens, geo):
        H, Hk, D, left, right, sinks, scale = geo
        B, N, _ = q.shape
        q, qa, qs = _lib.rows(q, H)
        k, ka, ks = _lib.rows(k, Hk)
        v, va, vs = _lib.rows(v, Hk)
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty(B, H, N, device=q.device, dtype=torch.float32)
        _lib.call("fta_window_attn_fwd", q.device, qa, qs, ka, ks, va, vs, _lib.DTYPE_CODES[q.dtype], B, H, Hk, N, D,
                  _lib.ptr(lens), left, right, sinks, scale, o.data_ptr(), _lib.dense_strides(q.shape, H),
                  lse.data_ptr())
        ctx.save_for_backward(q, k, v, o, lse, lens)
        ctx.geo = geo
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, do, _dlse):
        if do is None:
            return None, None, None, None, None
        q, k, v, o, lse, lens = ctx.saved_tensors
        H, Hk, D, left, right, sinks, scale = ctx.geo
        B, N, _ = q.shape
        q, qa, qs = _lib.rows(q, H)
        k, ka, ks = _lib.rows(k, Hk)
        v, va, vs = _lib.rows(v, Hk)
        do, da, ds = _lib.rows(do, H)
        dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
        sq, sk = _lib.dense_strides(q.shape, H), _lib.dense_strides(k.shape, Hk)
        nbytes = _lib.size_of("fta_window_attn_bwd_workspace_size", B, H, Hk, N, D, left, right, sinks)
        ws = _lib.workspace(nbytes, q.device)
        _lib.call("fta_window_attn_bwd", q.device, qa, qs, ka, ks, va, vs, o.data_ptr(), sq, da, ds,
                  _lib.DTYPE_CODES[q.dtype], B, H, Hk, N, D, _lib.ptr(lens), left, right, sinks, scale, lse.data_ptr(),
                  dq.data_ptr(), sq, dk.data_ptr(), sk, dv.data_ptr(), sk, ws.data_ptr(), nbytes)
        return dq, dk, dv, None, None


def flash_window_attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    num_heads: int,
    window: Tuple[int, int],
    num_sinks: int = 0,
    scale: Optional[float] = None,
    num_kv_heads: Optional[int] = None,
    seq_lens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Sliding-window attention with sinks (differentiable in q, k, v).

    Query i sees key j when ``j <= i + right`` and (``j >= i - left`` or
    ``j < num_sinks``): ``window=(w - 1, 0)`` is a causal window of w tokens, a window
    past the sequence plain causal or full attention, and the first ``num_sinks``
    tokens stay visible to every later query.

    Args:
        q: ``[B, N, num_heads * D]`` float16 or bfloat16, D a multiple of 16 up to 256.
        k, v: ``[B, N, num_kv_heads * D]``, the same type.
        window: ``(left, right)``, both >= 0.
        num_sinks: first tokens that stay visible.
        scale: softmax scale, default ``1 / sqrt(D)``; positive.
        num_kv_heads: grouped-query attention as in ``flash_sparse_attn``.
        seq_lens: int32 ``[B]`` on the device: tokens at or past it are padding.  They give
            o = 0, lse = -inf and zero gradients, and what q, k, v and the output's gradient
            hold there is not used.  Values outside ``[0, N]`` are clamped.  The tokens in
            front of it have to be finite (one that is not also reaches queries of the
            same tile that do not see it).

    Returns:
        ``(output [B, N, num_heads * D], lse [B, num_heads, N] float32 natural log)``; lse
        is not differentiable.

    Scores, softmax statistics and sums are float32; probabilities, and in the backward dS,
    are rounded to the inputs' type for the matrix units.  float16 gradients below 6e-5 lose
    bits: scale the loss.
    """
    what = "flash_window_attn"
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    num_heads, num_kv_heads, scale = _lib.scalars(what, num_heads, num_kv_heads, scale)
    geo = _geometry(what, q.shape, k.shape, v.shape, (q.dtype, k.dtype, v.dtype), num_heads, num_kv_heads,
                    tuple(_lib.whole(what, x) for x in window), _lib.whole(what, num_sinks), scale)
    _lib.check_device(what, q.device, k, v, seq_lens)
    if seq_lens is not None:
        if seq_lens.dtype != torch.int32 or seq_lens.shape != q.shape[:1]:
            raise ValueError(f"{what}: seq_lens must be int32 [B] = [{q.shape[0]}]")
        seq_lens = seq_lens.contiguous()
    return _WindowAttnFunc.apply(q, k, v, seq_lens, geo)


def flash_window_attn_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_lens: torch.Tensor,
    num_heads: int,
    window_left: int,
    num_sinks: int = 0,
    scale: Optional[float] = None,
    num_kv_heads: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``flash_window_attn`` with ``window=(window_left, 0)`` for the last T tokens of each
    request over its K/V cache.

    ``q`` is ``[B, T, num_heads * D]`` (T small: the T tokens and the query heads of a K/V
    head share each read of the cache), the caches ``[B, S, num_kv_heads * D]`` with rows
    16-byte aligned.  ``cache_lens`` (int32 ``[B]`` on the device, not read by the host)
    counts the cached tokens with these T (``flash_qk_norm_rope_append`` writes them);
    values outside ``[0, S]`` are clamped.  Token t stands at ``p = cache_lens[b] - T + t``
    and sees key j when ``j <= p`` and (``j >= p - window_left`` or ``j < num_sinks``);
    one that sees nothing (an idle request) gives o = 0, lse = -inf.  Cache rows that no
    token sees may hold anything.  ``window_left >= S`` is plain causal attention over the
    cache.  Probabilities are rounded to the inputs' type, as in ``flash_window_attn``.  Not
    differentiable.

    Returns ``(output [B, T, num_heads * D], lse [B, num_heads, T] float32)``.
    """
    what = "flash_window_attn_decode"
    window_left, num_sinks = _lib.whole(what, window_left), _lib.whole(what, num_sinks)
    if window_left < 0 or num_sinks < 0:
        raise ValueError(f"{what}: window_left and num_sinks must be non-negative")
    return cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, None, None,
                      min(window_left, _MAX), min(num_sinks, _MAX), scale)


__all__ = ["flash_window_attn", "flash_window_attn_decode"]
