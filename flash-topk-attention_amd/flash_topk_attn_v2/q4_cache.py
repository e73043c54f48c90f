"""K/V caches in 4 bits (HIP, gfx950): new tokens prepared and written into them in one
pass, attention of new tokens over them, and reading them back.

No counterpart in the reference.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from .qk_prep import _check, check_lens, offsets, written

_MAX = (1 << 30) - 1  # windows past this are the same as this


class Q4Cache(NamedTuple):
    """Keys and values of a batch in 4 bits (``flash_q4_cache`` makes an empty one).

    A row is one head of one token: groups of 32 columns (the last one filled up with
    zeros), each with a float16 scale d and a code n = 0 .. 15 per column, which stands for
    ``d * (n - 8)``.  Eight codes make a little-endian 32-bit word: column ``8 o + i`` of
    group g is bits ``4 i .. 4 i + 3`` of word ``4 g + o`` of a value row, and of word
    ``o * groups + g`` of a key row.

    ``k_codes`` and ``v_codes`` are uint8 ``[B, num_kv_heads, S, 16 * groups]``,
    ``k_scales`` and ``v_scales`` float16 ``[B, num_kv_heads, S, groups]``; the rows of a
    head follow each other, the codes of heads start at 16-byte steps and, where there is an
    even number of groups, their scales at 4-byte steps.
    """

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def flash_q4_cache(batch: int, tokens: int, num_kv_heads: int, head_dim: int, device) -> Q4Cache:
    """An empty ``Q4Cache`` (every row zero) for ``tokens`` tokens of ``batch`` requests."""
    what = "flash_q4_cache"
    B, S, Hk, D = (_lib.whole(what, x) for x in (batch, tokens, num_kv_heads, head_dim))
    if min(B, S, Hk, D) <= 0 or D % 16 != 0 or D > 256:
        raise ValueError(f"{what}: sizes must be positive, head_dim a multiple of 16 up to 256")
    groups = -(-D // 32)
    return Q4Cache(*(torch.zeros(B, Hk, S, n, device=device, dtype=t)
                     for n, t in ((16 * groups, torch.uint8), (groups, torch.float16)) * 2))


@lru_cache(maxsize=1024)
def _layout(what, shapes, strides, types, B, Hk, groups):
    """``(rows S, the strides that the library takes of each tensor of a Q4Cache, distances between the tensors that
    check_q4_written has passed)``, checked (calls of one shape are checked once)."""
    S = shapes[0][2] if len(shapes[0]) == 4 else 0
    widths = (16 * groups, groups) * 2
    names = Q4Cache._fields
    if types != (torch.uint8, torch.float16) * 2:
        raise ValueError(f"{what}: a 4-bit cache has uint8 codes and float16 scales")
    _lib.int_sizes(what, S)
    found = []
    for name, shape, stride, w in zip(names, shapes, strides, widths):
        if tuple(shape) != (B, Hk, S, w) or S == 0:
            raise ValueError(f"{what}: {name} must be {[B, Hk, 'S', w]}")
        sb, sh = stride[0] if B > 1 else 0, stride[1] if Hk > 1 else 0
        step = 15 if name.endswith("codes") else 1 - groups % 2  # bytes; elements, two where rows are read by pairs
        if (w > 1 and stride[3] != 1) or (S > 1 and stride[2] != w) or (sb | sh) & step:
            raise ValueError(f"{what}: the rows of a head of {name} must follow each other, heads at aligned steps")
        found.append(_lib.i64arr((sb, sh)))
    return S, tuple(found), set()


def _scale_step(groups):
    """Address bits that scales have clear: they are read by pairs where a row has an even number of them."""
    return 1 if groups % 2 else 3


def q4_args(what, cache, B, Hk, D, device, write=False):
    """``(S, address and strides of the four tensors)`` of a ``Q4Cache``, checked; with ``write`` by ``check_q4_written`` too."""
    if not isinstance(cache, Q4Cache):
        raise ValueError(f"{what}: cache must be a Q4Cache")
    kc, ks, vc, vs = cache
    groups = -(-D // 32)
    S, (kcs, kss, vcs, vss), apart = _layout(what, (kc.shape, ks.shape, vc.shape, vs.shape),
                                             (kc.stride(), ks.stride(), vc.stride(), vs.stride()),
                                             (kc.dtype, ks.dtype, vc.dtype, vs.dtype), B, Hk, groups)
    _lib.check_device(what, device, kc, ks, vc, vs)
    _lib.no_grad_inputs(what, ks, vs)
    kca, ksa, vca, vsa = kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr()
    if (kca | vca) & 15 or (ksa | vsa) & _scale_step(groups):
        raise ValueError(f"{what}: the cache's codes must be 16-byte aligned, its scales 4-byte where there is an even number of groups")
    if write:
        distances = (ksa - kca, vca - kca, vsa - kca)
        if distances not in apart:
            check_q4_written(what, cache)
            if len(apart) >= 1024:
                apart.clear()
            apart.add(distances)
    return S, (kca, kcs, ksa, kss, vca, vcs, vsa, vss)


@lru_cache(maxsize=1024)
def _q4_meet(shapes, strides, at):
    """Whether two rows of the four tensors share memory."""
    for (B, Hk, S, w), st in zip(shapes, strides):
        if _lib._rows_meet((B, Hk, S * w), (st[0], st[1], 1), 0):
            return True
    tensors = [*zip(shapes, strides, (1, 2) * 2)]
    return any(_lib.tensors_meet(tensors[i], tensors[j], at[j] - at[i]) for j in range(4) for i in range(j))


def check_q4_written(what: str, cache: Q4Cache) -> None:
    """Refuses caches whose rows share memory: what they would hold depends on which of two writes is the last."""
    at = tuple(t.data_ptr() for t in cache)
    if _q4_meet(tuple(t.shape for t in cache), tuple(t.stride() for t in cache), tuple(a - min(at) for a in at)):
        raise ValueError(f"{what}: rows of the cache share memory (an expanded cache, or tensors that overlap)")


def flash_qk_norm_rope_append_q4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cache: Q4Cache,
    cache_lens: torch.Tensor,
    num_heads: int,
    cos: torch.Tensor,
    sin: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    num_kv_heads: Optional[int] = None,
    position_offset: Union[int, torch.Tensor] = 0,
    interleaved: bool = False,
) -> torch.Tensor:
    """``flash_qk_norm_rope_append`` into a cache of 4-bit keys and values.

    The prepared keys (rounded to k's type) and the values are held in 4 bits: the scale of a
    group of 32 columns is its value of largest magnitude over -8 (of two equal ones the
    negative; rounded to float16, at most 65504 in magnitude), a column's code
    ``round(x / scale) + 8``, ties to even, held to 0 .. 15.  A column is off by at most half
    a scale, a sixteenth of its group's largest magnitude, but for values near the largest
    one's opposite, which are off by up to a whole scale and a 256th of it.  Where the largest
    magnitude is below 2^-11 (4.9e-4) the scale is a subnormal float16, off by up to 2^-25
    itself, and a column by up to 2^-22 (2.4e-7) more; groups of magnitudes up to 2^-22
    are held as zeros.  Values must be finite: infinities and NaN leave finite
    values of no meaning in their group.  Other arguments as for ``flash_qk_norm_rope_append``.  Not
    differentiable.

    Returns the prepared q ``[B, T, num_heads * D]``, which is not quantized.
    """
    what = "flash_qk_norm_rope_append_q4"
    _lib.no_grad_inputs(what, q, k, v, q_weight, k_weight)
    H, Hk, D, R, wt = _check(what, q, k, num_heads, num_kv_heads, cos, sin, q_weight, k_weight, eps)
    B, T, _ = q.shape
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError(f"{what}: v must have k's shape and type")
    check_lens(what, cache_lens, B)
    _lib.check_device(what, q.device, v, cache_lens)
    S, args = q4_args(what, cache, B, Hk, D, q.device, write=True)
    offset, offs = offsets(what, position_offset, B, q.device, cos.shape[0], S)
    q, qa, qs = _lib.rows(q, H)
    k, ka, ks = _lib.rows(k, Hk)
    v, va, vs = _lib.rows(v, Hk)
    qw, kw = (None if w is None else _lib.flat(w) for w in (q_weight, k_weight))
    cos, sin, lens = _lib.flat(cos), _lib.flat(sin), cache_lens.contiguous()
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    _lib.call("fta_qk_norm_rope_append_q4", q.device, qa, qs, ka, ks, va, vs, _lib.DTYPE_CODES[q.dtype], B, H, Hk, T, D,
              _lib.ptr(qw), _lib.ptr(kw), wt, cos.data_ptr(), sin.data_ptr(), cos.shape[0], R, offset, _lib.ptr(offs),
              float(eps), int(bool(interleaved)), lens.data_ptr(), S, qo.data_ptr(), _lib.dense_strides(q.shape, H), *args)
    written(*cache)
    return qo


def flash_q4_cache_read(cache: Q4Cache, head_dim: int, dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """What a 4-bit cache holds, in float16 or bfloat16 (each value rounded once): keys and
    values ``[B, S, num_kv_heads * head_dim]``, every row of the cache."""
    what = "flash_q4_cache_read"
    if not isinstance(cache, Q4Cache):
        raise ValueError(f"{what}: cache must be a Q4Cache")
    D = _lib.whole(what, head_dim)
    if D <= 0 or D % 16 != 0 or D > 256:
        raise ValueError(f"{what}: head_dim must be a multiple of 16 up to 256")
    if dtype not in _lib.HALVES:
        raise ValueError(f"{what}: dtype must be float16 or bfloat16")
    if not cache.k_codes.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    if cache.k_codes.ndim != 4 or 0 in cache.k_codes.shape:
        raise ValueError(f"{what}: k_codes must be [B, num_kv_heads, S, W], not empty")
    B, Hk = cache.k_codes.shape[:2]
    _lib.int_sizes(what, B, Hk)
    dev = cache.k_codes.device
    S, args = q4_args(what, cache, B, Hk, D, dev)
    k, v = (torch.empty(B, S, Hk * D, device=dev, dtype=dtype) for _ in range(2))
    _lib.call("fta_q4_read", dev, *args, _lib.DTYPE_CODES[dtype], B, Hk, S, D, k.data_ptr(), v.data_ptr())
    return k, v


@lru_cache(maxsize=1024)
def _geometry(what, q, dtype, num_heads, num_kv_heads, scale):
    if len(q) != 3:
        raise ValueError(f"{what}: q must be [B, T, num_heads * D]")
    if dtype not in _lib.HALVES:
        raise ValueError(f"{what}: q must be float16 or bfloat16")
    B, T, C = q
    H, Hk, D = _lib.head_counts(what, C, num_heads, num_kv_heads)
    if B == 0 or T == 0:
        raise ValueError(f"{what}: empty batch or no new tokens")
    _lib.int_sizes(what, B, T)
    return H, Hk, D, _lib.softmax_scale(what, scale, D)


def flash_window_attn_decode_q4(
    q: torch.Tensor,
    cache: Q4Cache,
    cache_lens: torch.Tensor,
    num_heads: int,
    window_left: int,
    num_sinks: int = 0,
    scale: Optional[float] = None,
    num_kv_heads: Optional[int] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """``flash_window_attn_decode`` over a cache of 4-bit keys and values.

    ``cache`` is a ``Q4Cache`` of ``[B, num_kv_heads, S]`` rows; the other arguments, which
    keys a token sees, rows that see nothing (o = 0, lse = -inf) and unseen rows (which may
    hold anything) as there.  The codes are multiplied as they stand, scales are applied
    in float32; probabilities times the values' scales are rounded to 8 bits of mantissa in
    bfloat16, to 16 in float16.  Made for few new tokens: from about 128 on,
    ``flash_q4_cache_read`` and a 16-bit attention take less time.  Not differentiable.

    Returns ``(output [B, T, num_heads * D], lse [B, num_heads, T] float32)``.
    """
    what = "flash_window_attn_decode_q4"
    window_left, num_sinks = _lib.whole(what, window_left), _lib.whole(what, num_sinks)
    if window_left < 0 or num_sinks < 0:
        raise ValueError(f"{what}: window_left and num_sinks must be non-negative")
    left, sinks = min(window_left, _MAX), min(num_sinks, _MAX)
    if not q.is_cuda:
        raise ValueError(f"{what} requires CUDA tensors")
    _lib.no_grad_inputs(what, q)
    num_heads, num_kv_heads, scale = _lib.scalars(what, num_heads, num_kv_heads, scale)
    H, Hk, D, scale = _geometry(what, q.shape, q.dtype, num_heads, num_kv_heads, scale)
    B, T, _ = q.shape
    dev = q.device
    check_lens(what, cache_lens, B)
    _lib.check_device(what, dev, cache_lens)
    S, args = q4_args(what, cache, B, Hk, D, dev)
    nbytes = _lib.size_of("fta_q4_attn_workspace_size", B, H, Hk, T, S, D, left, sinks)
    q, qa, qs = _lib.rows(q, H)
    lens = cache_lens.contiguous()
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(B, H, T, device=dev, dtype=torch.float32)
    ws = _lib.workspace(nbytes, dev) if nbytes else None
    _lib.call("fta_q4_attn", dev, qa, qs, *args, _lib.DTYPE_CODES[q.dtype], B, H, Hk, T, S, D, lens.data_ptr(), left, sinks,
              scale, o.data_ptr(), _lib.dense_strides(q.shape, H), lse.data_ptr(), _lib.ptr(ws), nbytes)
    return o, lse


__all__ = ["Q4Cache", "flash_q4_cache", "flash_q4_cache_read", "flash_qk_norm_rope_append_q4", "flash_window_attn_decode_q4"]
