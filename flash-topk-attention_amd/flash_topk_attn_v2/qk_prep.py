"""Queries and keys in front of scoring and attention (HIP, gfx950): the norm of
every head and the rotation by position in one pass, with its backward, and the
serving form that writes the new K and V rows into their caches.

No counterpart in the reference, whose callers prepare q and k by separate torch
operations.
"""

from __future__ import annotations

import warnings
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib


@lru_cache(maxsize=1024)
def _geometry(what, q, k, dtypes, cos, sin, table_types, q_weight, k_weight, weight_types, num_heads, num_kv_heads, eps):
    """``(H, Hk, D, R, weights' type code)`` from shapes and types, checked (calls of one
    shape are checked once)."""
    if len(q) != 3 or len(k) != 3:
        raise ValueError(f"{what}: q and k must be [B, N, heads * D]")
    if dtypes[0] not in _lib.HALVES or dtypes[1] != dtypes[0]:
        raise ValueError(f"{what}: q and k must both be float16 or bfloat16")
    H, Hk, D = _lib.head_counts(what, q[2], num_heads, num_kv_heads)
    if tuple(k) != (q[0], q[1], Hk * D):
        raise ValueError(f"{what}: k must be {[q[0], q[1], Hk * D]}")
    if q[0] == 0 or q[1] == 0:
        raise ValueError(f"{what}: empty batch or sequence")
    _lib.int_sizes(what, q[0], q[1], *cos)
    if len(cos) != 2 or cos != sin or table_types != (torch.float32, torch.float32):
        raise ValueError(f"{what}: cos and sin must be float32 tables [P, R / 2] of one shape")
    R = 2 * cos[1]
    if R <= 0 or R % 16 != 0 or R > D:
        raise ValueError(f"{what}: the rotated columns ({R}) must be a positive multiple of 16 up to D ({D})")
    if cos[0] == 0:
        raise ValueError(f"{what}: cos and sin have no rows")
    for w in (q_weight, k_weight):
        if w is not None and tuple(w) != (D,):
            raise ValueError(f"{what}: weights must be [D] = [{D}]")
    types = {t for t in weight_types if t is not None}
    if len(types) > 1 or not types <= set(_lib.DTYPE_CODES):
        raise ValueError(f"{what}: weights must both be float32, float16 or bfloat16")
    if not 0.0 < eps <= 3.0e38:
        raise ValueError(f"{what}: eps must be positive and a float32")
    return H, Hk, D, R, _lib.DTYPE_CODES[types.pop()] if types else _lib.DTYPE_F32


def _check(what, q, k, num_heads, num_kv_heads, cos, sin, qw, kw, eps):
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    num_heads, num_kv_heads, eps = _lib.scalars(what, num_heads, num_kv_heads, eps)
    geo = _geometry(what, q.shape, k.shape, (q.dtype, k.dtype), cos.shape, sin.shape, (cos.dtype, sin.dtype),
                    None if qw is None else qw.shape, None if kw is None else kw.shape,
                    (None if qw is None else qw.dtype, None if kw is None else kw.dtype), num_heads, num_kv_heads, eps)
    if cos.requires_grad or sin.requires_grad:
        raise ValueError(f"{what}: cos and sin are not differentiable")
    _lib.check_device(what, q.device, k, cos, sin, qw, kw)
    return geo


@lru_cache(maxsize=1024)
def _warn_of_short_tables(what, P, S, offset):
    """The lengths are on the device, so a position without a table row can only be foreseen:
    once per geometry."""
    if offset < 0 or S + offset > P:
        warnings.warn(f"{what}: cos and sin have rows for positions 0 .. {P - 1}, rows of the cache stand at {offset} .. "
                      f"{S + offset - 1}: tokens outside the tables are turned as the nearest row", stacklevel=3)


class _QKNormRopeFunc(torch.autograd.Function):
    """Autograd function behind ``flash_qk_norm_rope``."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, geo, eps, interleaved):
        H, Hk, D, R, wt = geo
        B, N, _ = q.shape
        q, qa, qs = _lib.rows(q, H)
        k, ka, ks = _lib.rows(k, Hk)
        qw, kw = (None if w is None else _lib.flat(w) for w in (q_weight, k_weight))
        qo, ko = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
        _lib.call("fta_qk_norm_rope", q.device, qa, qs, ka, ks, _lib.DTYPE_CODES[q.dtype], B, H, Hk, N, D, _lib.ptr(qw),
                  _lib.ptr(kw), wt, cos.data_ptr(), sin.data_ptr(), cos.shape[0], R, _lib.ptr(positions),
                  0 if positions is None else positions.stride(0), eps, interleaved, qo.data_ptr(),
                  _lib.dense_strides(q.shape, H), ko.data_ptr(), _lib.dense_strides(k.shape, Hk))
        ctx.save_for_backward(q, k, qw, kw, cos, sin, positions)
        ctx.args = geo, eps, interleaved
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dqo, dko):
        q, k, qw, kw, cos, sin, positions = ctx.saved_tensors
        (H, Hk, D, R, wt), eps, interleaved = ctx.args
        B, N, _ = q.shape
        dev = q.device
        q, qa, qs = _lib.rows(q, H)
        k, ka, ks = _lib.rows(k, Hk)
        dqo, dqa, dqs = _lib.rows(dqo, H)
        dko, dka, dks = _lib.rows(dko, Hk)
        dq, dk = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
        dqw = torch.empty(D, device=dev, dtype=qw.dtype) if qw is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty(D, device=dev, dtype=kw.dtype) if kw is not None and ctx.needs_input_grad[3] else None
        ws, nbytes = None, 0
        if dqw is not None or dkw is not None:
            nbytes = _lib.size_of("fta_qk_norm_rope_bwd_workspace_size", B, H, Hk, N, D)
            ws = _lib.workspace(nbytes, dev)
        _lib.call("fta_qk_norm_rope_bwd", dev, qa, qs, ka, ks, dqa, dqs, dka, dks, _lib.DTYPE_CODES[q.dtype], B, H, Hk, N,
                  D, _lib.ptr(qw), _lib.ptr(kw), wt, cos.data_ptr(), sin.data_ptr(), cos.shape[0], R,
                  _lib.ptr(positions), 0 if positions is None else positions.stride(0), eps, interleaved, dq.data_ptr(),
                  _lib.dense_strides(q.shape, H), dk.data_ptr(), _lib.dense_strides(k.shape, Hk), _lib.ptr(dqw),
                  _lib.ptr(dkw), _lib.ptr(ws), nbytes)
        return dq, dk, dqw, dkw, None, None, None, None, None, None


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
    (differentiable in q, k and the weights).  A head whose output's gradient is zero, as
    behind ``seq_lens`` of ``flash_window_attn``, adds nothing to any gradient, whatever
    it holds.

    Args:
        q: ``[B, N, num_heads * D]`` float16 or bfloat16, D a multiple of 16 up to 256.
        k: ``[B, N, num_kv_heads * D]``, the same type.
        cos, sin: float32 tables ``[P, R / 2]`` of the angles of positions ``0 .. P - 1``;
            the first ``R`` columns of a head are turned, ``R`` a multiple of 16 up to D.
            Tables that are not contiguous are copied at every call.
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
    geo = _check(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps)
    B, N, _ = q.shape
    if positions is None:
        if N > cos.shape[0]:
            raise ValueError(f"{what}: cos and sin have {cos.shape[0]} rows for {N} tokens")
    else:
        _lib.check_device(what, q.device, positions)
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: positions must be int32 or int64")
        if positions.shape not in ((N,), (B, N)):
            raise ValueError(f"{what}: positions must be [N] or [B, N] = {[B, N]}")
        if positions.dtype == torch.int64:  # into the tables' range first: the narrow type would wrap
            positions = positions.clamp(0, cos.shape[0] - 1).to(torch.int32)
        positions = positions.contiguous().expand(B, N)
    return _QKNormRopeFunc.apply(q, k, q_weight, k_weight, _lib.flat(cos), _lib.flat(sin), positions, geo, float(eps),
                                 int(bool(interleaved)))


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
    16-byte aligned; no two rows, of one cache or of both, may share memory, and q, k and v
    may lie in them only where a row is written to itself).  ``cache_lens`` (int32 ``[B]`` on the device, not read by the host)
    counts each request's cached tokens with these T: token t is written to row
    ``cache_lens[b] - T + t`` and turned as position ``row + position_offset`` (the
    length of a shared prefix, for instance).  Rows outside ``[0, S)`` are not written.
    Positions outside the tables take their nearest row, which turns those tokens wrongly; a
    call whose cache has such rows (tables of fewer than ``S + position_offset``) warns once.
    Other arguments as for ``flash_qk_norm_rope``.  Not differentiable.

    Returns the prepared q ``[B, T, num_heads * D]``.
    """
    what = "flash_qk_norm_rope_append"
    _lib.no_grad_inputs(what, q, k, v, q_weight, k_weight, k_cache, v_cache)
    H, Hk, D, R, wt = _check(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps)
    B, T, _ = q.shape
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type")
    check_cache(what, q, k_cache, v_cache, cache_lens, B, Hk * D)
    _lib.check_device(what, q.device, v)
    kca, kcs = _lib.rows_in_place(what, k_cache, Hk)
    vca, vcs = _lib.rows_in_place(what, v_cache, Hk)
    _lib.check_written(what, k_cache, v_cache)
    position_offset = _lib.whole(what, position_offset)
    if not -(1 << 31) <= position_offset < (1 << 31):
        raise ValueError(f"{what}: position_offset out of range")
    _warn_of_short_tables(what, cos.shape[0], k_cache.shape[1], position_offset)
    q, qa, qs = _lib.rows(q, H)
    k, ka, ks = _lib.rows(k, Hk)
    v, va, vs = _lib.rows(v, Hk)
    qw, kw = (None if w is None else _lib.flat(w) for w in (q_weight, k_weight))
    cos, sin, lens = _lib.flat(cos), _lib.flat(sin), cache_lens.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    _lib.call("fta_qk_norm_rope_append", q.device, qa, qs, ka, ks, va, vs, _lib.DTYPE_CODES[q.dtype], B, H, Hk, T, D,
              _lib.ptr(qw), _lib.ptr(kw), wt, cos.data_ptr(), sin.data_ptr(), cos.shape[0], R, position_offset,
              float(eps), int(bool(interleaved)), lens.data_ptr(), k_cache.shape[1], qo.data_ptr(),
              _lib.dense_strides(q.shape, H), kca, kcs, vca, vcs)
    for c in (k_cache, v_cache):
        if not c.is_inference():  # written in place (inference tensors keep no version)
            torch.autograd.graph.increment_version(c)
    return qo


def check_cache(what, q, k_cache, v_cache, cache_lens, B, width):
    """Shapes, types and devices of a pair of caches and their lengths."""
    shape = k_cache.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != width or shape[1] == 0:
        raise ValueError(f"{what}: k_cache must be [B, S, num_kv_heads * D] = [{B}, S, {width}]")
    _lib.int_sizes(what, shape[1])
    if v_cache.shape != shape:
        raise ValueError(f"{what}: v_cache must have k_cache's shape")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError(f"{what}: the caches must have q's type")
    if cache_lens.dtype != torch.int32 or cache_lens.shape != (B,):
        raise ValueError(f"{what}: cache_lens must be int32 [B] = [{B}]")
    _lib.check_device(what, q.device, k_cache, v_cache, cache_lens)


__all__ = ["flash_qk_norm_rope", "flash_qk_norm_rope_append"]
