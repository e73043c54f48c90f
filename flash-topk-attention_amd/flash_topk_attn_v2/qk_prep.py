"""Queries and keys in front of scoring and attention (HIP, gfx950): the norm of
every head and the rotation by position in one pass, with its backward, and the
serving form that writes the new K and V rows into their caches.

No counterpart in the reference, whose callers prepare q and k by separate torch
operations.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib


def _check_common(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps):
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError(f"{what}: q and k must be [B, N, heads * D]")
    if q.device.type != "cuda":
        raise ValueError(f"{what} requires CUDA tensors")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must both be float16 or bfloat16")
    H, Hk, D = _lib.head_counts(what, q.shape[2], num_heads, num_kv_heads)
    if tuple(k.shape) != (q.shape[0], q.shape[1], Hk * D):
        raise ValueError(f"{what}: k must be {[q.shape[0], q.shape[1], Hk * D]}")
    if q.shape[0] == 0 or q.shape[1] == 0:
        raise ValueError(f"{what}: empty batch or sequence")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"{what}: cos and sin must be float32 tables [P, R / 2] of one shape")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"{what}: cos and sin are not differentiable")
    R = 2 * cos.shape[1]
    if R <= 0 or R % 16 != 0 or R > D:
        raise ValueError(f"{what}: the rotated columns ({R}) must be a positive multiple of 16 up to D ({D})")
    if cos.shape[0] == 0:
        raise ValueError(f"{what}: cos and sin have no rows")
    dtypes = {w.dtype for w in (q_weight, k_weight) if w is not None}
    if len(dtypes) > 1 or not dtypes <= {torch.float32, torch.float16, torch.bfloat16}:
        raise ValueError(f"{what}: weights must both be float32, float16 or bfloat16")
    for w in (q_weight, k_weight):
        if w is not None and tuple(w.shape) != (D,):
            raise ValueError(f"{what}: weights must be [D] = [{D}]")
    if not 0.0 < float(eps) < float("inf"):
        raise ValueError(f"{what}: eps must be positive")
    _lib.check_tensors(what, q.device, k=k, cos=cos, sin=sin, q_weight=q_weight, k_weight=k_weight)
    return H, Hk, D, R


def _table(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _weights(q_weight, k_weight):
    """Contiguous weights and the code of their type."""
    codes = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
    w = [None if x is None else x.contiguous() for x in (q_weight, k_weight)]
    return w[0], w[1], next((codes[x.dtype] for x in w if x is not None), _lib.DTYPE_F32)


def _dense(B, N, heads, D):
    return _lib.i64arr((N * heads * D, D, heads * D))


class _QKNormRopeFunc(torch.autograd.Function):
    """Autograd function behind ``flash_qk_norm_rope``."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, H, Hk, eps, interleaved):
        B, N, C = q.shape
        D, dev = C // H, q.device
        qq, qs = _lib.token_view(q, "bnc", H)
        kk, ks = _lib.token_view(k, "bnc", Hk)
        qw, kw, wt = _weights(q_weight, k_weight)
        qo = torch.empty(B, N, C, device=dev, dtype=q.dtype)
        ko = torch.empty(B, N, Hk * D, device=dev, dtype=q.dtype)
        with _lib.on_device(dev):
            rc = _lib.lib().fta_qk_norm_rope(
                _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(kk), _lib.i64arr(ks), _lib.dtype_code(q.dtype), B, H, Hk, N, D,
                _lib.ptr(qw), _lib.ptr(kw), wt, _lib.ptr(cos), _lib.ptr(sin), cos.shape[0], 2 * cos.shape[1],
                _lib.ptr(positions), 0 if positions is None else positions.stride(0), eps, int(interleaved),
                _lib.ptr(qo), _dense(B, N, H, D), _lib.ptr(ko), _dense(B, N, Hk, D), _lib.stream_ptr(dev))
        _lib.check(rc, "flash_qk_norm_rope")
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.args = H, Hk, eps, interleaved
        return qo, ko

    @staticmethod
    def backward(ctx, dqo, dko):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        H, Hk, eps, interleaved = ctx.args
        B, N, C = q.shape
        D, dev = C // H, q.device
        qq, qs = _lib.token_view(q, "bnc", H)
        kk, ks = _lib.token_view(k, "bnc", Hk)
        dqq, dqs = _lib.token_view(dqo, "bnc", H)
        dkk, dks = _lib.token_view(dko, "bnc", Hk)
        qw, kw, wt = _weights(q_weight, k_weight)
        dq = torch.empty(B, N, C, device=dev, dtype=q.dtype)
        dk = torch.empty(B, N, Hk * D, device=dev, dtype=q.dtype)
        dqw = torch.empty_like(qw) if qw is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(kw) if kw is not None and ctx.needs_input_grad[3] else None
        need = dqw is not None or dkw is not None
        ws = _lib.workspace(_lib.size_of("fta_qk_norm_rope_bwd_workspace_size", B, H, Hk, N, D), dev) if need else None
        with _lib.on_device(dev):
            rc = _lib.lib().fta_qk_norm_rope_bwd(
                _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(kk), _lib.i64arr(ks), _lib.ptr(dqq), _lib.i64arr(dqs),
                _lib.ptr(dkk), _lib.i64arr(dks), _lib.dtype_code(q.dtype), B, H, Hk, N, D, _lib.ptr(qw), _lib.ptr(kw),
                wt, _lib.ptr(cos), _lib.ptr(sin), cos.shape[0], 2 * cos.shape[1], _lib.ptr(positions),
                0 if positions is None else positions.stride(0), eps, int(interleaved), _lib.ptr(dq),
                _dense(B, N, H, D), _lib.ptr(dk), _dense(B, N, Hk, D), _lib.ptr(dqw), _lib.ptr(dkw), _lib.ptr(ws),
                0 if ws is None else ws.numel(), _lib.stream_ptr(dev))
        _lib.check(rc, "flash_qk_norm_rope backward")
        return dq, dk, dqw, dkw, None, None, None, None, None, None, None


def flash_qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    num_heads: int,
    cos: torch.Tensor,
    sin: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    num_kv_heads: Optional[int] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every query and key head and rotation by position, in one pass
    (differentiable in q, k and the weights).

    Args:
        q: ``[B, N, num_heads * D]`` float16 or bfloat16, D a multiple of 16 up to 256.
        k: ``[B, N, num_kv_heads * D]``, the same type.
        cos, sin: float32 tables ``[P, R / 2]`` of the angles of positions ``0 .. P - 1``;
            the first ``R`` columns of a head are turned, ``R`` a multiple of 16 up to D.
        q_weight, k_weight: norm weights ``[D]`` (float32, float16 or bfloat16), or None for ones.
        eps: added to the mean square.
        num_kv_heads: heads of k, default ``num_heads``.
        positions: ``[B, N]`` or ``[N]`` int32 / int64, default each token's index.  Values
            outside ``[0, P)`` are taken as the nearest row of the tables.
        interleaved: turn columns ``(2i, 2i + 1)`` instead of ``(i, i + R / 2)``.

    Returns:
        The prepared ``(q, k)``, shapes and type of the inputs.
    """
    what = "flash_qk_norm_rope"
    H, Hk, D, R = _check_common(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps)
    B, N = q.shape[:2]
    if positions is None:
        if N > cos.shape[0]:
            raise ValueError(f"{what}: cos and sin have {cos.shape[0]} rows for {N} tokens")
    else:
        _lib.check_tensors(what, q.device, positions=positions)
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: positions must be int32 or int64")
        if tuple(positions.shape) not in ((N,), (B, N)):
            raise ValueError(f"{what}: positions must be [N] or [B, N] = {[B, N]}")
        if positions.dtype == torch.int64:  # into the tables' range first: the narrow type would wrap
            positions = positions.clamp(0, cos.shape[0] - 1).to(torch.int32)
        positions = positions.contiguous().expand(B, N)
    return _QKNormRopeFunc.apply(q, k, q_weight, k_weight, _table(cos), _table(sin), positions, H, Hk, float(eps),
                                 bool(interleaved))


def _check_cache(what, k_cache, v_cache, cache_lens, B, Hk, D, q):
    if k_cache.ndim != 3 or k_cache.shape[0] != B or k_cache.shape[2] != Hk * D or k_cache.shape[1] == 0:
        raise ValueError(f"{what}: k_cache must be [B, S, num_kv_heads * D] = [{B}, S, {Hk * D}]")
    if v_cache.shape != k_cache.shape:
        raise ValueError(f"{what}: v_cache must have k_cache's shape")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{what}: the caches must have q's type")
    if cache_lens.dtype != torch.int32 or tuple(cache_lens.shape) != (B,):
        raise ValueError(f"{what}: cache_lens must be int32 [B] = [{B}]")
    _lib.check_tensors(what, q.device, k_cache=k_cache, v_cache=v_cache, cache_lens=cache_lens)


def _cache_strides(what, c, D):
    """Strides of a cache that is read or written in place."""
    if c.stride(2) != 1 or c.data_ptr() % 16 != 0 or (c.stride(0) | c.stride(1)) & 7:
        raise ValueError(f"{what}: cache rows must be contiguous and 16-byte aligned")
    return _lib.i64arr((c.stride(0), D, c.stride(1)))


def _no_grad_inputs(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{what} is not differentiable: call it under torch.no_grad()")


def flash_qk_norm_rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_lens: torch.Tensor,
    num_heads: int,
    cos: torch.Tensor,
    sin: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    num_kv_heads: Optional[int] = None,
    position_offset: int = 0,
    interleaved: bool = False,
) -> torch.Tensor:
    """``flash_qk_norm_rope`` of the T new tokens of each request, their keys and values
    written into the caches in the same pass.

    ``q`` is ``[B, T, num_heads * D]``, ``k`` and ``v`` ``[B, T, num_kv_heads * D]``,
    the caches ``[B, S, num_kv_heads * D]`` (any batch and token stride that keeps rows
    16-byte aligned).  ``cache_lens`` (int32 ``[B]`` on the device, not read by the host)
    counts each request's cached tokens with these T: token t is written to row
    ``cache_lens[b] - T + t`` and turned as position ``row + position_offset`` (the
    length of a shared prefix, for instance).  Rows outside ``[0, S)`` are not written.
    Other arguments as for ``flash_qk_norm_rope``.  Not differentiable.

    Returns the prepared q ``[B, T, num_heads * D]``.
    """
    what = "flash_qk_norm_rope_append"
    _no_grad_inputs(what, q, k, v, q_weight, k_weight, k_cache, v_cache)
    H, Hk, D, R = _check_common(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps)
    B, T, C = q.shape
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type")
    _check_cache(what, k_cache, v_cache, cache_lens, B, Hk, D, q)
    _lib.check_tensors(what, q.device, v=v)
    if any(c.stride(0) == 0 and B > 1 for c in (k_cache, v_cache)) or any(
            c.stride(1) == 0 and c.shape[1] > 1 for c in (k_cache, v_cache)):
        raise ValueError(f"{what}: the caches must not be expanded")
    if not -(1 << 31) <= int(position_offset) < (1 << 31):
        raise ValueError(f"{what}: position_offset out of range")
    dev = q.device
    qq, qs = _lib.token_view(q, "bnc", H)
    kk, ks = _lib.token_view(k, "bnc", Hk)
    vv, vs = _lib.token_view(v, "bnc", Hk)
    qw, kw, wt = _weights(q_weight, k_weight)
    cos, sin, lens = _table(cos), _table(sin), cache_lens.contiguous()
    kcs, vcs = _cache_strides(what, k_cache, D), _cache_strides(what, v_cache, D)
    qo = torch.empty(B, T, C, device=dev, dtype=q.dtype)
    with _lib.on_device(dev):
        rc = _lib.lib().fta_qk_norm_rope_append(
            _lib.ptr(qq), _lib.i64arr(qs), _lib.ptr(kk), _lib.i64arr(ks), _lib.ptr(vv), _lib.i64arr(vs),
            _lib.dtype_code(q.dtype), B, H, Hk, T, D, _lib.ptr(qw), _lib.ptr(kw), wt, _lib.ptr(cos), _lib.ptr(sin),
            cos.shape[0], R, int(position_offset), float(eps), int(bool(interleaved)), _lib.ptr(lens),
            k_cache.shape[1], _lib.ptr(qo), _dense(B, T, H, D), _lib.ptr(k_cache), kcs, _lib.ptr(v_cache), vcs,
            _lib.stream_ptr(dev))
    _lib.check(rc, what)
    torch.autograd.graph.increment_version((k_cache, v_cache))
    return qo


__all__ = ["flash_qk_norm_rope", "flash_qk_norm_rope_append"]
