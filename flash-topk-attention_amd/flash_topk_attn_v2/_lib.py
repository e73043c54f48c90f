"""ctypes binding of libfta_gfx950.so (the C ABI declared in include/fta.h).

The library is the only compute path: there is no CPU or PyTorch fallback.  If
the shared object is missing or a call fails, an exception is raised.
"""

from __future__ import annotations

import ctypes
import os
from functools import lru_cache
from typing import Sequence

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libfta_gfx950.so")

FTA_OK = 0
FTA_ERR_ARG = 1
FTA_ERR_UNSUPPORTED = 2
FTA_ERR_HIP = 3
DTYPE_BF16 = 0
DTYPE_F16 = 1
DTYPE_F32 = 2  # norm weights only

_p = ctypes.c_void_p
_i = ctypes.c_int
_i64 = ctypes.c_int64
_f = ctypes.c_float
_sz = ctypes.c_size_t
_i64p = ctypes.POINTER(ctypes.c_int64)

_SIGNATURES = {
    "fta_last_error": (ctypes.c_char_p, []),
    "fta_version": (_i, []),
    "fta_block_score_workspace_size": (_sz, [_i, _i, _i, _i]),
    "fta_block_score": (_i, [_p, _p, _i, _i, _i, _i, _i, _i64p, _i64p, _i, _i, _i, _f, _p, _p, _sz, _p]),
    "fta_block_score_lse": (_i, [_p, _p, _i, _i, _i, _i, _i, _i64p, _i64p, _i, _i, _i, _f, _p, _p, _p]),
    "fta_topk_select": (_i, [_p, _i64, _i, _i64, _i64, _i, _i, _i, _i, _f, _p, _p, _p, _p]),
    "fta_topk_score_workspace_size": (_sz, [_i, _i, _i, _i]),
    "fta_topk_score": (_i, [_p, _p, _i, _i, _i, _i, _i, _i64p, _i64p, _i, _i, _i, _f, _i, _f, _p, _p, _p, _p,
                            _sz, _p]),
    "fta_topk_score_candidates": (_i, [_p, _p, _i, _i, _i, _i, _i, _i64p, _i64p, _i, _i, _i, _f, _i, _p, _sz, _p]),
    "fta_topk_select_candidates": (_i, [_p, _p, _i, _i, _i, _i, _i, _i64p, _i64p, _i, _i, _i, _f, _i, _f, _p, _p,
                                        _p, _p, _sz, _p]),
    "fta_topk_score_workspace_size_ex": (_sz, [_i] * 8),
    "fta_topk_score_workspace_min": (_sz, [_i] * 8),
    "fta_qblock_merge": (_i, [_p, _p, _i64, _i, _i, _i, _i, _p, _p, _p, _p]),
    "fta_qblock_merge_maxid": (_i, [_p, _p, _i64, _i, _i, _p, _i, _p, _p, _p, _p]),
    "fta_qblock_union": (_i, [_p, _i, _i, _i, _i, _i, _i, _i, _p, _p, _p]),
    "fta_build_reverse_indices_workspace_size": (_sz, [_i, _i, _i, _i]),
    "fta_build_reverse_indices": (_i, [_p, _p, _i, _i, _i, _i, _i, _p, _p, _p, _p, _sz, _p]),
    "fta_sort_by_count": (_i, [_p, _i64, _p, _p, _p]),
    "fta_sparse_attn_fwd_workspace_size": (_sz, [_i] * 10),
    "fta_sparse_attn_fwd_splits": (_i, [_i] * 10),
    "fta_sparse_attn_fwd": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _p, _i, _i, _i, _i, _i, _i,
                                 _i, _i, _f, _p, _i64p, _p, _p, _sz, _p]),
    "fta_sparse_attn_fwd_gqa": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _i, _i, _i, _i,
                                     _i, _i, _i, _i, _f, _p, _i64p, _p, _p, _sz, _p]),
    "fta_preprocess_delta": (_i, [_p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _p, _p]),
    "fta_sparse_attn_bwd_workspace_size": (_sz, [_i] * 10),
    "fta_sparse_attn_bwd": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _p, _i, _i, _i,
                                 _i, _i, _i, _i, _i, _f, _p, _p, _p, _i64p, _p, _i64p, _p, _i64p, _p, _sz, _p]),
    "fta_sparse_attn_bwd_gqa": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _i,
                                     _i, _i, _i, _i, _i, _i, _i, _f, _p, _p, _p, _i64p, _p, _i64p, _p, _i64p, _p,
                                     _sz, _p]),
    "fta_sparse_attn_bwd_dq": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _i, _i,
                                    _i, _i, _i, _i, _i, _i, _f, _p, _p, _p, _i64p, _p]),
    "fta_sparse_attn_bwd_dkv": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _i,
                                     _i, _i, _i, _i, _i, _i, _i, _f, _p, _p, _p, _i64p, _p, _i64p, _p, _sz, _p]),
    "fta_sparse_attn_bwd_noalloc": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p,
                                         _i, _i, _i, _i, _i, _i, _i, _i, _f, _p, _p, _p, _i64p, _p, _i64p, _p,
                                         _i64p, _p]),
    "fta_qk_norm_rope": (_i, [_p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _p, _i, _p, _p, _i, _i, _p, _i64, _f,
                              _i, _p, _i64p, _p, _i64p, _p]),
    "fta_qk_norm_rope_bwd_workspace_size": (_sz, [_i] * 5),
    "fta_qk_norm_rope_bwd": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _p, _i, _p,
                                  _p, _i, _i, _p, _i64, _f, _i, _p, _i64p, _p, _i64p, _p, _p, _p, _sz, _p]),
    "fta_qk_norm_rope_append": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _p, _i, _p, _p, _i,
                                     _i, _i, _f, _i, _p, _i, _p, _i64p, _p, _i64p, _p, _i64p, _p]),
    "fta_window_attn_fwd": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p, _i, _i, _i, _f, _p,
                                 _i64p, _p, _p]),
    "fta_window_attn_bwd_workspace_size": (_sz, [_i] * 8),
    "fta_window_attn_bwd": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _p,
                                 _i, _i, _i, _f, _p, _p, _i64p, _p, _i64p, _p, _i64p, _p, _sz, _p]),
    "fta_cache_attn_workspace_size": (_sz, [_i] * 9),
    "fta_cache_attn": (_i, [_p, _i64p, _p, _i64p, _p, _i64p, _i, _i, _i, _i, _i, _i, _i, _p, _p, _i64p, _p, _i64p, _i,
                            _i, _i, _f, _p, _i64p, _p, _p, _sz, _p]),
}


class FtaError(RuntimeError):
    """A libfta call failed (launch error or unsupported configuration)."""


@lru_cache(maxsize=None)
def lib() -> ctypes.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} not found: build it with `python flash-topk-attention_amd/build_lib.py` "
            "(hipcc --offload-arch=gfx950). There is no non-HIP fallback."
        )
    so = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(so, name)
        fn.restype = res
        fn.argtypes = args
    return so


def check(rc: int, what: str) -> None:
    if rc == FTA_OK:
        return
    msg = lib().fta_last_error().decode(errors="replace")
    if rc == FTA_ERR_ARG:
        raise ValueError(f"{what}: {msg}")
    if rc == FTA_ERR_UNSUPPORTED:
        raise NotImplementedError(f"{what}: {msg}")
    raise FtaError(f"{what}: {msg}")


def stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


@lru_cache(maxsize=1024)
def size_of(name: str, *geometry: int) -> int:
    """A ``*_workspace_size`` of the library: a pure function of the geometry, so
    repeated calls of one shape skip the ctypes call."""
    return int(getattr(lib(), name)(*geometry))


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


@lru_cache(maxsize=1024)
def _i64const(vals: tuple):
    return (ctypes.c_int64 * len(vals))(*vals)


def i64arr(vals: Sequence[int]):
    """Constant int64 array (strides); equal values share one, which the library only reads."""
    return _i64const(tuple(map(int, vals)))


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return DTYPE_BF16
    if dt == torch.float16:
        return DTYPE_F16
    raise ValueError(f"unsupported dtype {dt}; expected bfloat16 or float16")


def call(name: str, device: torch.device, *args) -> None:
    """One entry point of the library, launched on ``device``'s current stream (appended as
    the last argument); a failure raises as ``check`` does."""
    fn = getattr(lib(), name)
    if device.index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:  # launches go to the current device
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != FTA_OK:
        check(rc, name)


@lru_cache(maxsize=4096)
def dense_strides(shape: tuple, heads: int):
    """Strides of a contiguous ``[B, N, heads * D]`` tensor as the library takes them."""
    _, N, C = shape
    return i64arr((N * C, C // heads, C))


@lru_cache(maxsize=4096)
def _row_strides(shape: tuple, stride: tuple, heads: int):
    """``{stride_b, stride_h, stride_n}`` of a ``[B, N, heads * D]`` tensor, or None where its
    rows are not contiguous or not whole 16-byte steps apart."""
    B, N, C = shape
    sb = stride[0] if B > 1 else 0
    sn = stride[1] if N > 1 else C
    if stride[2] != 1 or (sb | sn) & 7:
        return None
    return i64arr((sb, C // heads, sn))


def rows(x: torch.Tensor, heads: int):
    """``(tensor, address, strides)`` that address ``x`` ``[B, N, heads * D]`` by 16-byte
    loads; a copy only where its layout or its address does not allow them."""
    strides, at = _row_strides(x.shape, x.stride(), heads), x.data_ptr()
    if strides is None or at & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        strides, at = _row_strides(x.shape, x.stride(), heads), x.data_ptr()
    return x, at, strides


def rows_in_place(what: str, x: torch.Tensor, heads: int):
    """``(address, strides)`` of a tensor that is used where it is (a cache)."""
    strides, at = _row_strides(x.shape, x.stride(), heads), x.data_ptr()
    if strides is None or at & 15:
        raise ValueError(f"{what}: cache rows must be contiguous and 16-byte aligned")
    return at, strides


@lru_cache(maxsize=4096)
def _rows_meet(shape: tuple, stride: tuple, delta: int) -> bool:
    """Whether a row of ``[B, N, C]`` and one of the same layout ``delta`` elements on share an
    element (``delta`` 0: two different rows of the one)."""
    (B, N, C), (sb, sn, _) = shape, stride
    for db in range(1 - B, B):
        x = delta + db * sb
        near = -x // sn if sn else 0  # the token distances that bring the rows closest
        for ds in (near, near + 1):
            ds = min(max(ds, 1 - N), N - 1)
            if abs(x + ds * sn) < C and (delta or db or ds):
                return True
    return False


@lru_cache(maxsize=4096)
def _caches_meet(shape: tuple, k_stride: tuple, v_stride: tuple, delta: int) -> bool:
    """Whether two rows of a pair of caches ``[B, N, C]``, v ``delta`` elements behind k, share
    an element (layouts that differ and lie within each other are taken to)."""
    if _rows_meet(shape, k_stride, 0) or _rows_meet(shape, v_stride, 0):
        return True
    k_end, v_end = (sum((n - 1) * s for n, s in zip(shape, st)) for st in (k_stride, v_stride))
    if delta > k_end or -delta > v_end:
        return False
    dims = [i for i, n in enumerate(shape) if n > 1]
    return any(k_stride[i] != v_stride[i] for i in dims) or _rows_meet(shape, k_stride, delta) or delta == 0


def check_written(what: str, k: torch.Tensor, v: torch.Tensor) -> None:
    """Refuses caches whose rows share memory: what they would hold depends on which of two
    writes is the last."""
    if _caches_meet(k.shape, k.stride(), v.stride(), (v.data_ptr() - k.data_ptr()) // k.element_size()):
        raise ValueError(f"{what}: rows of the caches share memory (an expanded cache, or one that overlaps the other)")


def flat(x: torch.Tensor) -> torch.Tensor:
    """``x`` contiguous and 16-byte aligned (a table or weights)."""
    if x.is_contiguous() and x.data_ptr() & 15 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def check_device(what: str, device: torch.device, *tensors) -> None:
    """Every given tensor has to be on ``device`` (None is skipped)."""
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: a tensor is on {t.device}, expected {device}")


def head_counts(what: str, width: int, num_heads: int, num_kv_heads):
    """``(H, Hk, D)`` of a ``[..., H * D]`` tensor, checked."""
    H = int(num_heads)
    if H <= 0 or width % H != 0 or width == 0:
        raise ValueError(f"{what}: C ({width}) must be a positive multiple of num_heads ({H})")
    Hk = H if num_kv_heads is None else int(num_kv_heads)
    if Hk <= 0 or H % Hk != 0:
        raise ValueError(f"{what}: num_heads ({H}) must be a positive multiple of num_kv_heads ({Hk})")
    D = width // H
    if D % 16 != 0 or D > 256:
        raise ValueError(f"{what}: D ({D}) must be a multiple of 16 up to 256")
    return H, Hk, D


def int_sizes(what: str, *sizes: int) -> None:
    """Refuses sizes that the library's 32-bit ints do not hold (ctypes would wrap them)."""
    if max(sizes) >= 1 << 31:
        raise NotImplementedError(f"{what}: a size of {max(sizes)}; sizes must be below 2^31")


def whole(what: str, x) -> int:
    """``x`` as a Python integer; anything that is not a whole number is refused."""
    if type(x) is int:
        return x
    try:
        i = int(x)
    except (TypeError, ValueError, OverflowError):
        raise ValueError(f"{what}: {x!r} is not a whole number") from None
    if i != x:
        raise ValueError(f"{what}: {x!r} is not a whole number")
    return i


def scalars(what: str, num_heads, num_kv_heads, real):
    """Head counts and a real number as Python numbers: what a cached check may be keyed by."""
    return (whole(what, num_heads), None if num_kv_heads is None else whole(what, num_kv_heads),
            None if real is None else float(real))


HALVES = (torch.float16, torch.bfloat16)
DTYPE_CODES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16, torch.float32: DTYPE_F32}


SCALE_MAX = 2.0e38  # times log2(e) still a float32


def no_grad_inputs(what: str, *tensors) -> None:
    """Refuses a call whose gradients would be lost."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} is not differentiable: call it under torch.no_grad()")


def softmax_scale(what: str, scale, D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale <= SCALE_MAX:
        raise ValueError(f"{what}: scale must be positive and at most {SCALE_MAX}")
    return scale


def workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def token_view(x: torch.Tensor, layout: str, num_heads: int):
    """Return (tensor, [stride_b, stride_h, stride_n]) addressing x as [B][N][H][D]
    with unit D stride and 16-byte aligned rows; copies only when needed.

    layout "bnc": x is [B, N, H*D]; layout "bhnd": x is [B, H, N, D].
    """

    def ok(t, s0, s1, s2):
        return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and (s0 | s1 | s2) & 7 == 0

    if layout == "bnc":
        D = x.shape[2] // num_heads
        if not ok(x, x.stride(0), D, x.stride(1)):
            x = x.contiguous()
        return x, (x.stride(0), D, x.stride(1))
    if not ok(x, x.stride(0), x.stride(1), x.stride(2)):
        x = x.contiguous()
    return x, (x.stride(0), x.stride(1), x.stride(2))
