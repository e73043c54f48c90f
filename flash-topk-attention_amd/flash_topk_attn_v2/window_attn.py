"""Sliding-window attention with sinks (HIP, gfx950): the local layers beside the
top-k sparse ones, forward and backward, and its form for new tokens over K/V caches.

No counterpart in the reference.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from .cache_attn import cache_attn

_MAX = (1 << 30) - 1  # windows past this are the same as this


def _scale(what, scale, D):
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 3.0e38:
        raise ValueError(f"{what}: scale must be positive and finite")
    return scale


class _WindowAttnFunc(torch.autograd.Function):
    """Autograd function behind ``flash_window_attn``."""

    @staticmethod
    def forward(ctx, q, k, v, lens, H, Hk, left, right, sinks, scale):
        B, N, C = q.shape
        D, dev = C // H, q.device
        qq, qs = _lib.token_view(q, "bnc", H)
        kk, ks = _lib.token_view(k, "bnc", Hk)
        vv, vs = _lib.token_view(v, "bnc", Hk)
        o = torch.empty(B, N, C, device=dev, dtype=q.dtype)
        lse = torch.empty(B, H, N, device=dev, dtype=torch.float32)
        with _lib.on_device(dev):
            rc = _lib.lib().fta_window_attn_fwd(
                _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(kk), _lib.i64arr(ks), _lib.ptr(vv), _lib.i64arr(vs),
                _lib.dtype_code(q.dtype), B, H, Hk, N, D, _lib.ptr(lens), left, right, sinks, scale, _lib.ptr(o),
                _lib.i64arr((N * C, D, C)), _lib.ptr(lse), _lib.stream_ptr(dev))
        _lib.check(rc, "flash_window_attn")
        ctx.save_for_backward(q, k, v, o, lse, lens)
        ctx.args = H, Hk, left, right, sinks, scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, do, _dlse):
        q, k, v, o, lse, lens = ctx.saved_tensors
        H, Hk, left, right, sinks, scale = ctx.args
        B, N, C = q.shape
        D, dev = C // H, q.device
        qq, qs = _lib.token_view(q, "bnc", H)
        kk, ks = _lib.token_view(k, "bnc", Hk)
        vv, vs = _lib.token_view(v, "bnc", Hk)
        dd, ds = _lib.token_view(do, "bnc", H)
        dq = torch.empty(B, N, C, device=dev, dtype=q.dtype)
        dk = torch.empty(B, N, Hk * D, device=dev, dtype=q.dtype)
        dv = torch.empty(B, N, Hk * D, device=dev, dtype=q.dtype)
        sq, sk = _lib.i64arr((N * C, D, C)), _lib.i64arr((N * Hk * D, D, Hk * D))
        ws = _lib.workspace(_lib.size_of("fta_window_attn_bwd_workspace_size", B, H, Hk, N, D, left, right, sinks), dev)
        with _lib.on_device(dev):
            rc = _lib.lib().fta_window_attn_bwd(
                _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(kk), _lib.i64arr(ks), _lib.ptr(vv), _lib.i64arr(vs),
                _lib.ptr(o), sq, _lib.ptr(dd), _lib.i64arr(ds), _lib.dtype_code(q.dtype), B, H, Hk, N, D,
                _lib.ptr(lens), left, right, sinks, scale, _lib.ptr(lse), _lib.ptr(dq), sq, _lib.ptr(dk), sk,
                _lib.ptr(dv), sk, _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev))
        _lib.check(rc, "flash_window_attn backward")
        return dq, dk, dv, None, None, None, None, None, None, None


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
    """
    what = "flash_window_attn"
    if q.ndim != 3 or k.ndim != 3 or v.ndim != 3:
        raise ValueError(f"{what}: q, k and v must be [B, N, heads * D]")
    if q.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: q, k and v must all be float16 or all bfloat16")
    B, N, C = q.shape
    H, Hk, D = _lib.head_counts(what, C, num_heads, num_kv_heads)
    if B == 0 or N == 0:
        raise ValueError(f"{what}: empty batch or sequence")
    if tuple(k.shape) != (B, N, Hk * D) or tuple(v.shape) != (B, N, Hk * D):
        raise ValueError(f"{what}: k and v must be [B, N, num_kv_heads * D] = {[B, N, Hk * D]}")
    if len(window) != 2 or int(window[0]) < 0 or int(window[1]) < 0:
        raise ValueError(f"{what}: window must be (left, right), both non-negative")
    if int(num_sinks) < 0:
        raise ValueError(f"{what}: num_sinks must be non-negative")
    if seq_lens is not None and (seq_lens.dtype != torch.int32 or tuple(seq_lens.shape) != (B,)):
        raise ValueError(f"{what}: seq_lens must be int32 [B] = [{B}]")
    _lib.check_tensors(what, q.device, k=k, v=v, seq_lens=seq_lens)
    left, right, sinks = (min(int(x), _MAX) for x in (*window, num_sinks))
    lens = None if seq_lens is None else seq_lens.contiguous()
    return _WindowAttnFunc.apply(q, k, v, lens, H, Hk, left, right, sinks, _scale(what, scale, D))


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
    cache.  Not differentiable.

    Returns ``(output [B, T, num_heads * D], lse [B, num_heads, T] float32)``.
    """
    what = "flash_window_attn_decode"
    if int(window_left) < 0 or int(num_sinks) < 0:
        raise ValueError(f"{what}: window_left and num_sinks must be non-negative")
    return cache_attn(what, q, k_cache, v_cache, cache_lens, num_heads, num_kv_heads, None, None,
                      min(int(window_left), _MAX), min(int(num_sinks), _MAX), scale)


__all__ = ["flash_window_attn", "flash_window_attn_decode"]
