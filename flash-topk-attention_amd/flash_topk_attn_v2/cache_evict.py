"""Which rows of a K/V cache stay (HIP, gfx950): the attention that every cached key
receives, added up, and the eviction of the rows that received least.

No counterpart in the reference.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .q4_cache import _MAX, Q4Cache, _geometry, _layout, _q4_meet, _scale_step, q4_args
from .qk_prep import check_lens, written


@lru_cache(maxsize=1024)
def _weights_layout(what, shape, stride, dtype, B, Hk, write=True):
    """Strides of weights ``[B, Hk, S]``, checked (calls of one shape are checked once); rows that are written lie apart."""
    if len(shape) != 3 or tuple(shape[:2]) != (B, Hk) or shape[2] == 0 or dtype != torch.float32:
        raise ValueError(f"{what}: weights must be float32 [B, num_kv_heads, S] = [{B}, {Hk}, S]")
    _lib.int_sizes(what, shape[2])
    if shape[2] > 1 and stride[2] != 1:
        raise ValueError(f"{what}: the weights of a head must follow each other")
    if write and _lib._rows_meet(tuple(shape), (stride[0] if B > 1 else 0, stride[1] if Hk > 1 else 0, 1), 0):
        raise ValueError(f"{what}: rows of the weights share memory")
    return _lib.i64arr((stride[0] if B > 1 else 0, stride[1] if Hk > 1 else 0))


def flash_cache_weights(
    q: torch.Tensor,
    cache: Union[torch.Tensor, Q4Cache],
    lse: torch.Tensor,
    cache_lens: torch.Tensor,
    weights: torch.Tensor,
    num_heads: int,
    window_left: int,
    num_sinks: int = 0,
    scale: Optional[float] = None,
    num_kv_heads: Optional[int] = None,
) -> torch.Tensor:
    """Adds to ``weights`` the attention that every cached key receives from the last T tokens
    of its request: the sum over tokens and the query heads of its K/V head of
    ``exp(scale * q . k - lse)``.

    ``q`` ``[B, T, num_heads * D]`` and ``lse`` ``[B, num_heads, T]`` (float32) are those of the
    attention that ran: of ``flash_window_attn_decode``, its 4-bit form, or, with T the
    prompt's length, ``flash_window_attn`` with ``window=(window_left, 0)``.  ``cache`` is the
    keys, ``[B, S, num_kv_heads * D]`` of q's type with rows 16-byte aligned, or a
    ``Q4Cache``.  ``cache_lens`` (int32 ``[B]`` on the device, not read by the host) counts the
    cached tokens with these T; token t sees key j as in ``flash_window_attn_decode``; tokens
    that see nothing (lse = -inf) add nothing.  (Tokens are the last T of each request: prompts of
    different lengths that are padded behind their ends go one by one.)  ``weights`` is float32
    ``[B, num_kv_heads, S]``, written in place where ``j < cache_lens[b]``, and must overlap no
    other argument.  Unseen rows of the cache may hold anything.
    Sums are float32 in a fixed order.  Not differentiable.

    Returns ``weights``.
    """
    what = "flash_cache_weights"
    window_left, num_sinks = _lib.whole(what, window_left), _lib.whole(what, num_sinks)
    if window_left < 0 or num_sinks < 0:
        raise ValueError(f"{what}: window_left and num_sinks must be non-negative")
    left, sinks = min(window_left, _MAX), min(num_sinks, _MAX)
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _lib.no_grad_inputs(what, q, lse, weights)
    num_heads, num_kv_heads, scale = _lib.scalars(what, num_heads, num_kv_heads, scale)
    H, Hk, D, scale = _geometry(what, q.shape, q.dtype, num_heads, num_kv_heads, scale)
    B, T, _ = q.shape
    dev = q.device
    check_lens(what, cache_lens, B)
    if lse.dtype != torch.float32 or lse.shape != (B, H, T):
        raise ValueError(f"{what}: lse must be float32 [B, num_heads, T] = {[B, H, T]}")
    _lib.check_device(what, dev, lse, cache_lens, weights)
    ws_strides = _weights_layout(what, weights.shape, weights.stride(), weights.dtype, B, Hk)
    if isinstance(cache, Q4Cache):
        S, (ka, ks, sa, ss, *_) = q4_args(what, cache, B, Hk, D, dev)
    else:
        if not isinstance(cache, torch.Tensor) or cache.ndim != 3 or cache.shape[0] != B or cache.shape[2] != Hk * D or cache.shape[1] == 0:
            raise ValueError(f"{what}: cache must be keys [B, S, num_kv_heads * D] = [{B}, S, {Hk * D}] or a Q4Cache")
        if cache.dtype != q.dtype:
            raise ValueError(f"{what}: the keys must have q's type")
        _lib.check_device(what, dev, cache)
        _lib.no_grad_inputs(what, cache)
        S = cache.shape[1]
        _lib.int_sizes(what, S)
        (ka, ks), sa, ss = _lib.rows_in_place(what, cache, Hk), None, None
    if weights.shape[2] != S:
        raise ValueError(f"{what}: weights must be float32 [B, num_kv_heads, S] = {[B, Hk, S]}")
    _lib.check_apart(what, "weights", weights, q, lse, cache_lens, *(cache if isinstance(cache, Q4Cache) else (cache,)))
    nbytes = _lib.size_of("fta_cache_weights_workspace_size", B, H, Hk, T, S, D, left, sinks)
    q, qa, qs = _lib.rows(q, H)
    lens, lse = cache_lens.contiguous(), lse.contiguous()
    ws = _lib.workspace(nbytes, dev) if nbytes else None
    _lib.call("fta_cache_weights", dev, qa, qs, ka, ks, sa, ss, _lib.DTYPE_CODES[q.dtype], B, H, Hk, T, S, D,
              lens.data_ptr(), left, sinks, scale, lse.data_ptr(), weights.data_ptr(), ws_strides, _lib.ptr(ws), nbytes)
    written(weights)
    return weights


def _metas(tensors):
    return tuple((t.shape, t.stride(), t.dtype) for t in tensors)


@lru_cache(maxsize=1024)
def _moved_layout(what, q4, metas, B, Hk, budget, write):
    """``(rows S, byte strides {b, head, row} and row bytes of the cache's tensors, strides of the
    weights, places that _check_apart has passed)`` of a cache and its weights, checked (calls of one
    shape are checked once)."""
    *cache, (w_shape, w_stride, w_type) = metas
    found, nbytes = [], []
    if q4:
        shape = cache[1][0]
        groups = shape[3] if len(shape) == 4 else 0
        if not 1 <= groups <= 8:
            raise ValueError(f"{what}: k_scales must be [B, num_kv_heads, S, groups], up to 8 groups")
        S, strides, _ = _layout(what, *zip(*cache), B, Hk, groups)
        for (shape, _, dtype), st in zip(cache, strides):
            size = dtype.itemsize
            found += [size * st[0], size * st[1], size * shape[3]]
            nbytes.append(size * shape[3])
    else:
        (shape, _, dtype), (v_shape, _, v_type) = cache
        if len(shape) != 3 or shape[0] != B or 0 in shape or shape[2] % Hk != 0 or v_shape != shape:
            raise ValueError(f"{what}: the caches must both be [B, S, num_kv_heads * D], {B} requests and {Hk} heads")
        S, D = shape[1], shape[2] // Hk
        if D % 16 != 0 or D > 256:
            raise ValueError(f"{what}: D ({D}) must be a multiple of 16 up to 256")
        if dtype not in _lib.HALVES or v_type != dtype:
            raise ValueError(f"{what}: the caches must both be float16 or bfloat16")
        _lib.int_sizes(what, S)
        for shape, stride, _ in cache:
            st = _lib._row_strides(shape, stride, Hk)
            if st is None:
                raise ValueError(f"{what}: cache rows must be contiguous and 16-byte aligned")
            found += [2 * st[0], 2 * st[1], 2 * st[2]]
            nbytes.append(2 * D)
    w_strides = _weights_layout(what, w_shape, w_stride, w_type, B, Hk, write)
    if w_shape[2] != S:
        raise ValueError(f"{what}: weights must have the cache's {S} rows, not {w_shape[2]}")
    if budget > S:
        raise ValueError(f"{what}: budget ({budget}) must not pass the cache's rows ({S})")
    return S, _lib.i64arr(found), (ctypes.c_int32 * len(nbytes))(*nbytes), w_strides, set()


def _meet(a, b, delta):
    """Whether tensors of two of ``_metas``, the second ``delta`` bytes behind the first, share a byte."""
    (sa, ta, da), (sb, tb, db) = a, b
    return _lib.tensors_meet((sa, ta, da.itemsize), (sb, tb, db.itemsize), delta)


def _check_aligned(what, q4, nbytes, at):
    wide, scales = (at[0] | at[2], at[1] | at[3]) if q4 else (at[0] | at[1], 0)
    if wide & 15 or at[-1] & 3 or scales & _scale_step(nbytes[1] // 2):
        raise ValueError(f"{what}: cache rows must be 16-byte aligned (scales 4-byte where there is an even number of groups)")


def _check_apart(what, q4, metas, to_metas, at, to_at, in_place=False):
    """Refuses what is written where rows share memory, and ``out`` that overlaps the inputs."""
    *cache, _ = to_metas
    shapes, strides = tuple(m[0] for m in cache), tuple(m[1] for m in cache)
    if q4:
        if _q4_meet(shapes, strides, tuple(a - to_at[0] for a in to_at[:4])):
            raise ValueError(f"{what}: rows of the cache share memory (an expanded cache, or tensors that overlap)")
    elif _lib._caches_meet(shapes[0], strides[0], strides[1], (to_at[1] - to_at[0]) // 2):
        raise ValueError(f"{what}: rows of the caches share memory (an expanded cache, or one that overlaps the other)")
    if any(_meet(m, to_metas[-1], to_at[-1] - a) for m, a in zip(to_metas[:-1], to_at)):
        raise ValueError(f"{what}: the weights overlap the cache")
    if not in_place and any(_meet(m, n, b - a) for m, a in zip(metas, at) for n, b in zip(to_metas, to_at)):
        raise ValueError(f"{what}: out overlaps the inputs")


def flash_cache_evict(
    cache: Union[Tuple[torch.Tensor, torch.Tensor], Q4Cache],
    weights: torch.Tensor,
    cache_lens: torch.Tensor,
    budget: int,
    num_recent: int = 0,
    num_sinks: int = 0,
    out: Optional[tuple] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keeps at most ``budget`` rows of every request and K/V head of a cache: the first
    ``num_sinks``, the last ``num_recent`` and, of those between, the ones of largest
    ``weights`` (of equal ones the lower rows; NaN counts as less than any number).  Rows that
    stay keep their order and move to the front.

    ``cache`` is ``(k_cache, v_cache)``, ``[B, S, num_kv_heads * D]`` each, or a ``Q4Cache``;
    ``weights`` float32 ``[B, num_kv_heads, S]``, as ``flash_cache_weights`` adds them up;
    ``cache_lens`` int32 ``[B]`` on the device (not read by the host; values outside ``[0, S]``
    are clamped).  In place, or, with ``out = (cache, weights)`` of the same kind and at least
    ``budget`` rows, into those (``out`` must not overlap the inputs).  The weights move with
    their rows; behind them they are set to zero, up to the old length in place, to the end
    in ``out``.  Rows of the cache behind the new length are left as they are.  No two rows
    of what is written may share memory.

    A cache whose rows moved no longer holds token j at row j: the attention of new tokens
    takes distances in rows (``window_left >= S`` sees every row that stayed), and
    ``flash_qk_norm_rope_append`` takes the rows that went, ``cache_lens - new_lens`` added
    up, as its ``position_offset``.  Not differentiable.

    Returns ``(new_lens int32 [B] = min(cache_lens, budget), kept int32 [B, num_kv_heads,
    budget])``: the former row of each row, -1 behind the new length.  ``cache_lens`` is not
    changed.
    """
    what = "flash_cache_evict"
    budget, recent, sinks = (_lib.whole(what, x) for x in (budget, num_recent, num_sinks))
    if not weights.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    if weights.ndim != 3 or 0 in weights.shape:
        raise ValueError(f"{what}: weights must be float32 [B, num_kv_heads, S], not empty")
    if recent < 0 or sinks < 0 or budget <= 0 or recent + sinks > budget:
        raise ValueError(f"{what}: budget must be positive and num_recent + num_sinks fit in it")
    B, Hk, S = weights.shape
    dev = weights.device
    _lib.int_sizes(what, B, Hk, S, budget)
    check_lens(what, cache_lens, B)
    _lib.check_device(what, dev, cache_lens)
    q4 = isinstance(cache, Q4Cache)
    if not q4 and (not isinstance(cache, (tuple, list)) or len(cache) != 2 or not all(isinstance(t, torch.Tensor) for t in cache)):
        raise ValueError(f"{what}: cache must be (k_cache, v_cache) or a Q4Cache")
    tensors = (*cache, weights)
    if out is None:
        to = tensors
    elif not isinstance(out, (tuple, list)) or len(out) != 2 or not isinstance(out[0], Q4Cache if q4 else (tuple, list)) or len(
            out[0]) != len(cache):
        raise ValueError(f"{what}: out must be (cache, weights), a cache of the same kind")
    else:
        to = (*out[0], out[1])
        _lib.check_device(what, dev, *to)
        _lib.no_grad_inputs(what, *to)
    _lib.check_device(what, dev, *tensors)
    _lib.no_grad_inputs(what, *tensors)
    metas = _metas(tensors)
    S, strides, nbytes, w_strides, apart = _moved_layout(what, q4, metas, B, Hk, budget, out is None)
    at = [t.data_ptr() for t in tensors]
    _check_aligned(what, q4, nbytes, at)
    base = at[0]
    if out is None:
        to_metas, to_at = metas, at
        S_out, to_strides, to_w_strides = S, strides, w_strides
        places = tuple([a - base for a in at])
    else:
        to_metas, to_at = _metas(to), [t.data_ptr() for t in to]
        S_out, to_strides, to_bytes, to_w_strides, _ = _moved_layout(what, q4, to_metas, B, Hk, budget, True)
        _check_aligned(what, q4, to_bytes, to_at)
        places = to_metas, tuple([a - base for a in (*at, *to_at)])
        if to_metas[0][2] != metas[0][2] or list(to_bytes) != list(nbytes):
            raise ValueError(f"{what}: out must have the cache's type and head dim")
    if places not in apart:
        _check_apart(what, q4, metas, to_metas, at, to_at, out is None)
        if len(apart) >= 1024:
            apart.clear()
        apart.add(places)
    _lib.check_apart(what, "weights", to[-1], cache_lens)
    n = len(cache)
    lens = cache_lens.contiguous()
    new_lens = torch.empty(B, device=dev, dtype=torch.int32)
    kept = torch.empty(B, Hk, budget, device=dev, dtype=torch.int32)
    addresses = ctypes.c_void_p * n
    _lib.call("fta_cache_evict", dev, n, addresses(*at[:n]), strides, addresses(*to_at[:n]), to_strides, nbytes, at[n],
              w_strides, to_at[n], to_w_strides, B, Hk, S, S_out, budget, recent, sinks, lens.data_ptr(),
              new_lens.data_ptr(), kept.data_ptr())
    written(*to)
    return new_lens, kept


__all__ = ["flash_cache_weights", "flash_cache_evict"]
