"""Refusals of the operators around the sparse attention, without a GPU: the Python
checks raise before anything is launched, and the C entries return a status."""

import pytest
import torch

import flash_topk_attn_v2 as fta
from flash_topk_attn_v2 import _lib

BF = torch.bfloat16




def test_cpu_tensors_are_refused():
    x, t = torch.zeros(1, 4, 64, dtype=BF), torch.zeros(4, 32)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        fta.flash_qk_norm_rope(x, x, 1, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        fta.flash_qk_norm_rope_append(x, x, x, x, x, n, 1, t, t)
    with pytest.raises(ValueError, match="CUDA"):
        fta.flash_window_attn(x, x, x, 1, (3, 0))
    with pytest.raises(ValueError, match="CUDA"):
        fta.flash_window_attn_decode(x, x, x, n, 1, 3)
    with pytest.raises(ValueError, match="CUDA"):
        fta.flash_prefix_attn_decode(x, x[0], x[0], x, x, n, 1)
    with pytest.raises(ValueError, match="required"):
        fta.flash_prefix_attn_decode(x, None, None, x, x, n, 1)
    with pytest.raises(ValueError, match="non-negative"):
        fta.flash_window_attn_decode(x, x, x, n, 1, -1)


def _prep(L, B=1, H=2, Hk=1, N=4, D=64, P=4, R=64, dtype=0, wt=2, eps=1e-6, append=False, S=8):
    z = _lib.i64arr((0, 0, 0))
    if append:
        return L.fta_qk_norm_rope_append(None, z, None, z, None, z, dtype, B, H, Hk, N, D, None, None, wt, None, None, P, R,
                                         0, eps, 0, None, S, None, z, None, z, None, z, None)
    return L.fta_qk_norm_rope(None, z, None, z, dtype, B, H, Hk, N, D, None, None, wt, None, None, P, R, None, 0, eps, 0,
                              None, z, None, z, None)


@pytest.mark.parametrize("bad", [dict(B=0), dict(H=0), dict(N=0), dict(D=0), dict(D=24), dict(D=272), dict(R=8), dict(R=80),
                                 dict(R=0), dict(P=0), dict(dtype=2), dict(dtype=-1), dict(wt=3), dict(eps=0.0),
                                 dict(eps=float("nan"))])
@pytest.mark.parametrize("append", [False, True])
def test_prep_entry(bad, append):
    L = _lib.lib()
    assert _prep(L, append=append, **bad) == _lib.FTA_ERR_ARG
    assert L.fta_last_error()


def test_prep_entry_rows():
    L = _lib.lib()
    assert _prep(L, N=5, P=4) == _lib.FTA_ERR_ARG  # more tokens than table rows
    assert _prep(L, append=True, S=0) == _lib.FTA_ERR_ARG
    assert L.fta_qk_norm_rope_bwd_workspace_size(1, 2, 1, 4, 24) == 0
    assert L.fta_qk_norm_rope_bwd_workspace_size(1, 2, 1, 4, 64) > 0


def _window(L, B=1, H=4, Hk=2, N=10, D=64, left=3, right=0, sinks=0, scale=0.1, dtype=0):
    z = _lib.i64arr((0, 0, 0))
    return L.fta_window_attn_fwd(None, z, None, z, None, z, dtype, B, H, Hk, N, D, None, left, right, sinks, scale, None, z,
                                 None, None)


def _window_bwd(L, ws=0, **kw):
    z = _lib.i64arr((0, 0, 0))
    a = dict(B=1, H=4, Hk=2, N=10, D=64, left=3, right=0, sinks=0, scale=0.1, dtype=0) | kw
    return L.fta_window_attn_bwd(None, z, None, z, None, z, None, z, None, z, a["dtype"], a["B"], a["H"], a["Hk"], a["N"],
                                 a["D"], None, a["left"], a["right"], a["sinks"], a["scale"], None, None, z, None, z, None,
                                 z, None, ws, None)


BAD = [dict(B=0), dict(H=3), dict(Hk=0), dict(N=0), dict(N=-1), dict(D=8), dict(D=260), dict(left=-1), dict(right=-2),
       dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(dtype=2)]


@pytest.mark.parametrize("bad", BAD)
def test_window_entries(bad):
    L = _lib.lib()
    assert _window(L, **bad) == _lib.FTA_ERR_ARG
    assert _window_bwd(L, **bad) == _lib.FTA_ERR_ARG


def test_window_entry_sizes():
    L = _lib.lib()
    assert _window(L, N=(1 << 29) + 1) == _lib.FTA_ERR_UNSUPPORTED
    assert _window_bwd(L) == _lib.FTA_ERR_ARG  # no workspace
    assert b"workspace" in L.fta_last_error()
    # delta and the log2 lse, then fp32 dK / dV parts of small grids and of the sinks' tiles
    assert L.fta_window_attn_bwd_workspace_size(1, 4, 2, 10, 64, 3, 0, 0) >= 2 * 256
    big = (1, 32, 8, 32768, 128, 1023, 0)
    none, four = (L.fta_window_attn_bwd_workspace_size(*big, s) for s in (0, 4))
    assert none == 2 * 4 * 32 * 32768  # 4096 workgroups: no parts
    assert four > none and (four - none) % (2 * 8 * 64 * 128 * 4) == 0
    assert L.fta_window_attn_bwd_workspace_size(1, 4, 3, 10, 64, 3, 0, 0) == 0


def _cache(L, B=1, H=4, Hk=2, T=1, S=10, D=64, P=0, left=3, sinks=0, scale=0.1, dtype=0, ws=0):
    z = _lib.i64arr((0, 0, 0))
    return L.fta_cache_attn(None, z, None, z, None, z, dtype, B, H, Hk, T, S, D, None, None, z, None, z, P, left, sinks, scale,
                            None, z, None, None, ws, None)


@pytest.mark.parametrize("bad", [dict(B=0), dict(H=5), dict(Hk=-2), dict(T=0), dict(S=0), dict(D=12), dict(D=512), dict(P=-1),
                                 dict(left=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(dtype=7)])
def test_cache_entry(bad):
    L = _lib.lib()
    assert _cache(L, **bad) == _lib.FTA_ERR_ARG


def test_cache_entry_sizes():
    L = _lib.lib()
    assert _cache(L, P=5) == _lib.FTA_ERR_UNSUPPORTED  # a window behind a shared prefix
    assert _cache(L, S=(1 << 29) + 1) == _lib.FTA_ERR_UNSUPPORTED
    assert _cache(L, P=5, left=10) == _lib.FTA_ERR_ARG  # parts without a workspace
    assert L.fta_cache_attn_workspace_size(1, 4, 2, 1, 10, 64, 0, 3, 0) == 0  # one part: o written directly
    assert L.fta_cache_attn_workspace_size(1, 4, 2, 1, 10, 64, 70, 10, 0) > 0
    assert L.fta_cache_attn_workspace_size(1, 4, 3, 1, 10, 64, 0, 3, 0) == 0


def _pointers(entry):
    """Entry, its arguments as a list, and the places of the pointers it requires.  Every
    pointer is some address that nothing reads: with one of them null the entry returns
    before any launch."""
    L = _lib.lib()
    z, x = _lib.i64arr((0, 0, 0)), 4096
    if entry == "prep":
        args = [x, z, x, z, 0, 1, 2, 1, 4, 64, None, None, 2, x, x, 4, 64, None, 0, 1e-6, 0, x, z, x, z, None]
        return L.fta_qk_norm_rope, args, (0, 1, 2, 3, 13, 14, 21, 22, 23, 24)
    if entry == "prep_bwd":
        args = [x, z, x, z, x, z, x, z, 0, 1, 2, 1, 4, 64, None, None, 2, x, x, 4, 64, None, 0, 1e-6, 0, x, z, x, z,
                None, None, None, 0, None]
        return L.fta_qk_norm_rope_bwd, args, (*range(8), 17, 18, 25, 26, 27, 28)
    if entry == "append":
        args = [x, z, x, z, x, z, 0, 1, 2, 1, 4, 64, None, None, 2, x, x, 4, 64, 0, 1e-6, 0, x, 8, x, z, x, z, x, z, None]
        return L.fta_qk_norm_rope_append, args, (*range(6), 15, 16, 22, *range(24, 30))
    if entry == "window":
        args = [x, z, x, z, x, z, 0, 1, 4, 2, 10, 64, None, 3, 0, 0, 0.1, x, z, x, None]
        return L.fta_window_attn_fwd, args, (*range(6), 17, 18, 19)
    if entry == "window_bwd":
        size = L.fta_window_attn_bwd_workspace_size(1, 4, 2, 10, 64, 3, 0, 0)
        args = [x, z, x, z, x, z, x, z, x, z, 0, 1, 4, 2, 10, 64, None, 3, 0, 0, 0.1, x, x, z, x, z, x, z, x, size, None]
        return L.fta_window_attn_bwd, args, (*range(10), *range(21, 29))
    size = L.fta_cache_attn_workspace_size(1, 4, 2, 1, 10, 64, 5, 10, 0)
    args = [x, z, x, z, x, z, 0, 1, 4, 2, 1, 10, 64, x, x, z, x, z, 5, 10, 0, 0.1, x, z, x, x, size, None]
    return L.fta_cache_attn, args, (*range(6), *range(13, 18), *range(22, 26))


@pytest.mark.parametrize("entry", ["prep", "prep_bwd", "append", "window", "window_bwd", "cache"])
def test_null_pointers(entry):
    call, args, required = _pointers(entry)
    assert len(args) == len(call.argtypes)
    for i in required:
        assert call(*(args[:i] + [None] + args[i + 1:])) == _lib.FTA_ERR_ARG, i


def test_launch_limits():
    L = _lib.lib()
    assert L.fta_cache_attn_workspace_size(1 << 24, 1, 1, 1, 10, 64, 0, 3, 0) == 0  # 2^32 threads
    assert _cache(L, B=1 << 24, H=1, Hk=1) == _lib.FTA_ERR_UNSUPPORTED


def test_sizes_past_32_bits():
    """They are refused before they would wrap."""
    from flash_topk_attn_v2 import cache_attn, qk_prep, window_attn

    n, f = 1 << 31, torch.float32
    prep = ("prep", (1, n, 64), (1, n, 64), (BF, BF), (n, 32), (n, 32), (f, f), None, None, (None, None), 1, 1, 1e-6)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        qk_prep._geometry(*prep)
    with pytest.raises(NotImplementedError, match="2\\^31"):
        window_attn._geometry("window", (1, n, 64), (1, n, 64), (1, n, 64), (BF, BF, BF), 1, 1, (3, 0), 0, None)
    for S, P in ((n, 0), (4, n)):
        with pytest.raises(NotImplementedError, match="2\\^31"):
            cache_attn._geometry("cache", (1, 1, 64), BF, 1, 1, S, P, None, 0, None)


def test_window_workspace_of_many_sinks():
    """The parts of the sinks' walks stay a few hundred MB, however many sinks and sequences."""
    L = _lib.lib()
    for B, H, Hk, N, D, left, sinks in ((1, 32, 8, 32768, 128, 1023, 16384), (1, 32, 32, 32768, 256, 15, 8192),
                                        (64, 16, 16, 4096, 128, 63, 100), (8, 4, 1, 100000, 64, 0, 99000)):
        rows = 2 * 4 * B * H * N
        assert 0 < L.fta_window_attn_bwd_workspace_size(B, H, Hk, N, D, left, 0, sinks) <= rows + 512 + (300 << 20)
