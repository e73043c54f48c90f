"""Limits of the operators around the sparse attention that are checked without a GPU."""

import itertools
import warnings

import numpy as np
import pytest
import torch

import flash_topk_attn_v2 as fta
from flash_topk_attn_v2 import _lib, cache_attn, qk_prep, window_attn


@pytest.mark.parametrize("B,H,Hk,N,D", [(1 << 30, 4096, 4096, 1 << 29, 64), (1 << 30, 1 << 20, 1 << 16, 1 << 20, 64),
                                        ((1 << 31) - 1, 1 << 20, 1 << 20, 1 << 20, 256), (1 << 28, 1 << 16, 1, 1 << 19, 16)])
def test_sizes_whose_products_wrap(B, H, Hk, N, D):
    """Sizes of no real tensor: refused, where a 64-bit product wrapped to zero was divided by."""
    L, z, x = _lib.lib(), _lib.i64arr((0, 0, 0)), 4096  # an address that nothing reads
    assert L.fta_window_attn_bwd_workspace_size(B, H, Hk, N, D, 3, 0, 4) == 0
    assert L.fta_cache_attn_workspace_size(B, H, Hk, min(N, 1 << 20), 10, D, 0, 3, 0) == 0
    assert L.fta_qk_norm_rope_bwd_workspace_size(B, H, Hk, N, D) == 0
    rc = L.fta_window_attn_fwd(x, z, x, z, x, z, 0, B, H, Hk, N, D, None, 3, 0, 4, 0.1, x, z, x, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED
    rc = L.fta_cache_attn(x, z, x, z, x, z, 0, B, H, Hk, min(N, 1 << 20), 10, D, x, None, z, None, z, 0, 3, 0, 0.1, x, z, x,
                          None, 0, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED
    rc = L.fta_qk_norm_rope(x, z, x, z, 0, B, H, Hk, N, D, None, None, 2, x, x, N, 16, None, 0, 1e-6, 0, x, z, x, z, None)
    assert rc == _lib.FTA_ERR_UNSUPPORTED


@pytest.mark.parametrize("B,S,W,st", [(1, 1, 16, (0, 0)), (2, 3, 16, (48, 16)), (2, 3, 16, (96, 32)), (3, 2, 16, (32, 96)),
                                      (2, 3, 16, (48, 8)), (2, 3, 16, (40, 16)), (2, 3, 16, (0, 16)), (2, 3, 16, (48, 0)),
                                      (3, 4, 16, (16, 56)), (3, 4, 16, (160, 40)), (1, 4, 16, (8, 16)), (4, 1, 16, (16, 8))])
def test_rows_that_share_memory(B, S, W, st):
    """The rule that refuses caches whose rows share memory, against every pair of elements."""
    own = [{b * st[0] + s * st[1] + i for i in range(W)} for b in range(B) for s in range(S)]
    alone = sum(map(len, own)) == len(set().union(*own))
    for delta in range(-200, 201, 8):
        other = [{x + delta for x in row} for row in own]
        apart = alone and set().union(*own).isdisjoint(set().union(*other))
        assert _lib._caches_meet((B, S, W), (*st, 1), (*st, 1), delta) == (not apart), delta


def test_caches_of_the_usual_layouts():
    B, S, W = 3, 5, 32
    pairs = [torch.zeros(S, B, 2 * W).transpose(0, 1).split(W, -1), torch.zeros(B, S, 2, W).unbind(2),
             torch.zeros(B, 2, S, W).unbind(1), torch.zeros(2, B, S, W).unbind(0), (torch.zeros(B, S, W), torch.zeros(B, S, W)),
             torch.zeros(B, 2 * S, W).split(S, 1)]
    for pair in pairs:
        for k, v in itertools.permutations(pair):
            _lib.check_written("caches", k, v)
    one = torch.zeros(B, S, W)
    wide = torch.zeros(B, S, W + 16)
    for k, v in ((one, one), (one[:1].expand(B, -1, -1), torch.zeros(B, S, W)), (torch.zeros(B, S, W), one[:, :1].expand(-1, S, -1)),
                 (wide[..., :W], wide[..., 16:]), (torch.zeros(B, S + 1, W)[:, :-1], one.as_strided((B, S, W), (16, W, 1))),
                 (one, one.transpose(0, 1).reshape(B, S, W).as_strided((B, S, W), (W, W, 1)))):
        with pytest.raises(ValueError, match="share memory"):
            _lib.check_written("caches", k, v)
    with pytest.raises(ValueError, match="share memory"):  # rows of a cache moved by one token
        both = torch.zeros(B, S + 1, W)
        _lib.check_written("caches", both[:, :-1], both[:, 1:])


def test_tables_shorter_than_the_cache():
    """Warned of once per geometry; tables that hold every cached position are not."""
    check = qk_prep._warn_of_short_tables
    check.cache_clear()
    for P, S, offset in ((7, 8, 0), (107, 8, 100), (8, 8, -1), (1, 1, 1)):
        with pytest.warns(UserWarning, match="nearest row"):
            check("append", P, S, offset)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        check("append", 7, 8, 0)  # already said
        for P, S, offset in ((8, 8, 0), (108, 8, 100), (1, 1, 0), (1 << 20, 8, 5)):
            check("append", P, S, offset)


def test_fractions_are_not_sizes():
    """Sizes were cut to whole numbers: a window of 3.9 tokens was one of 3."""
    for x in (4, 4.0, np.int32(4), np.float64(4), torch.tensor(4), torch.tensor(4.0), True + 3):
        got = _lib.whole("sizes", x)
        assert type(got) is int and got == 4
    for x in (3.9, -0.5, float("nan"), float("inf"), np.float32(0.1), torch.tensor(1.5), None, "four"):
        with pytest.raises(ValueError, match="whole number"):
            _lib.whole("sizes", x)
    with pytest.raises(ValueError, match="whole number"):
        _lib.scalars("sizes", 4, 2.5, None)
    x, n = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for bad in (dict(window_left=3.5), dict(num_sinks=0.5)):  # refused in front of the look at the tensors
        with pytest.raises(ValueError, match="whole number"):
            fta.flash_window_attn_decode(x, x, x, n, 1, **(dict(window_left=3) | bad))


def test_reals_past_float32():
    """A scale whose product with log2(e) is infinite made every score NaN, an infinite eps every row zero."""
    BF, f = torch.bfloat16, torch.float32
    shape, table = (1, 4, 64), (4, 32)

    def prep(eps):
        return qk_prep._geometry("prep", shape, shape, (BF, BF), table, table, (f, f), None, None, (None, None), 1, None, eps)

    def window(scale):
        return window_attn._geometry("window", shape, shape, shape, (BF,) * 3, 1, None, (3, 0), 0, scale)

    def cache(scale):
        return cache_attn._geometry("cache", shape, BF, 1, None, 10, 0, 3, 0, scale)

    for x in (1e-30, 1.0, 1e30, 2e38):
        prep(x), window(x), cache(x)
    for call, bad in ((prep, 1e39), (prep, float("inf")), (window, 2.5e38), (window, 1e39), (cache, 2.5e38), (cache, 1e39)):
        with pytest.raises(ValueError, match="positive"):
            call(bad)
    L, z, x = _lib.lib(), _lib.i64arr((0, 0, 0)), 4096  # an address that nothing reads
    for v in (2.5e38, float("inf")):
        assert L.fta_window_attn_fwd(x, z, x, z, x, z, 0, 1, 1, 1, 4, 64, None, 3, 0, 0, v, None, z, x, None) == _lib.FTA_ERR_ARG
        assert b"scale" in L.fta_last_error()
        assert L.fta_cache_attn(x, z, x, z, x, z, 0, 1, 1, 1, 1, 10, 64, x, None, z, None, z, 0, 3, 0, v, None, z, x, None, 0,
                                None) == _lib.FTA_ERR_ARG
        assert b"scale" in L.fta_last_error()
    assert L.fta_qk_norm_rope(x, z, x, z, 0, 1, 1, 1, 4, 64, None, None, 2, x, x, 4, 64, None, 0, float("inf"), 0, None, z, x, z,
                              None) == _lib.FTA_ERR_ARG
    assert b"eps" in L.fta_last_error()
