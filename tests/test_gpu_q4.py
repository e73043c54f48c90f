"""Caches of 4-bit keys and values: what the append writes, what reading gives back, and the
attention over them, against their definitions in float64."""

import math

import pytest
import torch

import _operators_ref as R
import _q4_ref as Q
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _tables(P, R2, dev):
    a = torch.arange(P, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(R2, dtype=torch.float64) / R2)
    return a.cos().float().to(dev), a.sin().float().to(dev)


# dtype, B, T, S, H, Hk, D, rotated, interleaved, lens
APPEND = [
    (BF, 1, 1, 1, 1, 1, 64, 64, False, [1]),
    (FP, 2, 3, 50, 4, 2, 16, 16, False, [50, 2]),        # a row of half a group; tokens in front of the cache are dropped
    (BF, 3, 5, 33, 4, 4, 128, 128, False, [5, 33, 40]),   # the last past the cache
    (FP, 2, 40, 64, 6, 3, 80, 32, True, [40, 64]),
    (BF, 2, 7, 30, 8, 2, 256, 64, False, [7, 29]),
    (BF, 1, 2, 9, 5, 1, 96, 96, True, [9]),
    (FP, 2, 3, 11, 4, 2, 144, 128, False, [11, 3]),
    (BF, 1, 700, 700, 16, 16, 128, 128, False, [700]),   # five groups of rows a wave
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_append(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, B, T, S, H, Hk, D, rot, inter, lens = case
    say("append_q4", case)
    q, k, v = (rand((B, T, h * D), 5 + i, dtype, gpu) for i, h in enumerate((H, Hk, Hk)))
    qw, kw = (1 + 0.1 * rand((D,), 8 + i, torch.float32, gpu) for i in (0, 1))
    cos, sin = _tables(S + 10, rot // 2, gpu)
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    c = Q.cache(B, S, Hk, D, gpu, 1)
    was = [t.clone() for t in c]
    got = fta.flash_qk_norm_rope_append_q4(q, k, v, c, ln, H, cos, sin, qw, kw, num_kv_heads=Hk, position_offset=4,
                                           interleaved=inter)
    # the 16-bit append's rows, quantized: codes and scales are the same numbers
    kc, vc = (torch.zeros(B, S, Hk * D, device=gpu, dtype=dtype) for _ in range(2))
    q16 = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, ln, H, cos, sin, qw, kw, num_kv_heads=Hk, position_offset=4,
                                        interleaved=inter)
    assert torch.equal(got, q16)
    for x, key, codes, scales, old in ((kc, True, c.k_codes, c.k_scales, was[:2]), (vc, False, c.v_codes, c.v_scales, was[2:])):
        n, d = Q.quantize(x.view(B, S, Hk, D).transpose(1, 2))
        want = Q.pack(n, key)
        for b in range(B):
            new = torch.zeros(S, dtype=torch.bool, device=gpu)
            new[max(0, lens[b] - T):max(0, min(S, lens[b]))] = True
            assert torch.equal(codes[b][:, new], want[b][:, new]) and torch.equal(scales[b][:, new], d[b][:, new])
            assert torch.equal(codes[b][:, ~new], old[0][b][:, ~new]) and torch.equal(scales[b][:, ~new], old[1][b][:, ~new])
    # and near what they stand for: a code is off by half a scale, by a whole one where it is held to 15, and
    # the 16-bit rounding of k by its own half step
    pos = ln[:, None] - T + torch.arange(T, device=gpu)
    exact = R.turned(k.double(), Hk, kw.double(), cos, sin, pos + 4, 1e-6, inter).unflatten(-1, (Hk, D))
    val, step = (x.transpose(1, 2) for x in Q.values(c.k_codes, c.k_scales, True, D))
    for b in range(B):
        for t in range(T):
            at = lens[b] - T + t
            if 0 <= at < S:
                off = (val[b, at] - exact[b, t]).abs()
                assert (off <= step[b, at] * (1 + 2.0 ** -7) + 2 * R.half_step(dtype) * exact[b, t].abs() + 1e-6).all()


def test_borders_and_extremes(gpu):
    """Values at the borders between codes, equal largest magnitudes of both signs, zeros, tiny and huge groups."""
    import flash_topk_attn_v2 as fta

    D = 64
    rows = []
    for top in (8.0, -8.0):
        rows.append([top] + [x * 0.5 for x in range(-15, 16)] + [0.0] * 32)       # every half: ties to even
    rows.append([3.0, -3.0] + [1.5] * 30 + [-5.0, 5.0] + [2.5] * 30)               # the negative one is -8
    rows.append([0.0] * 64)
    rows.append([1e-7, -1e-7] * 16 + [3e-7] * 32)                                   # below and around the smallest scale
    rows.append([3.0e38, 1.0e30] * 16 + [-7e5] + [5e5] * 31)                        # scales held to 65504
    for dtype in (BF, FP):
        v = torch.tensor(rows, dtype=torch.float64).clamp(*(((-6e4, 6e4)) if dtype == FP else (-3.3e38, 3.3e38)))
        v = v.to(dtype).to(gpu)[None]  # [1, rows, D]
        T = v.shape[1]
        cos, sin = _tables(T, 32, gpu)
        c = fta.flash_q4_cache(1, T, 1, D, gpu)
        fta.flash_qk_norm_rope_append_q4(v, v, v, c, torch.tensor([T], dtype=torch.int32, device=gpu), 1, cos, sin)
        n, d = Q.quantize(v)
        assert torch.equal(c.v_scales[0], d) and torch.equal(c.v_codes[0], Q.pack(n, False))


@pytest.mark.parametrize("D", [16, 64, 80, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_read(gpu, D, dtype):
    import flash_topk_attn_v2 as fta

    B, S, Hk = 3, 37, 2
    c = Q.cache(B, S, Hk, D, gpu, 2)
    k, v = fta.flash_q4_cache_read(c, D, dtype)
    for got, key, codes, scales in ((k, True, c.k_codes, c.k_scales), (v, False, c.v_codes, c.v_scales)):
        want = Q.values(codes, scales, key, D)[0].to(dtype).transpose(1, 2).flatten(-2)
        assert got.shape == (B, S, Hk * D) and torch.equal(got, want)


# dtype, B, T, H, Hk, D, S, left, sinks, lens
DECODE = [
    (BF, 1, 1, 1, 1, 64, 1, 0, 0, [1]),
    (BF, 4, 1, 8, 2, 128, 100, 20, 4, [100, 1, 0, 57]),
    (FP, 3, 2, 4, 4, 64, 333, 100, 0, [333, 200, 64]),
    (BF, 2, 1, 8, 1, 256, 700, 10000, 3, [700, 129]),
    (FP, 2, 5, 16, 2, 80, 300, 31, 33, [3, 300]),       # fewer tokens than new ones: rows that see nothing; 40 rows
    (BF, 1, 1, 32, 8, 128, 3000, 2047, 4, [3000]),      # many parts
    (BF, 1, 1, 2, 2, 64, 9000, 8191, 100, [8999]),
    (FP, 70, 1, 8, 8, 128, 257, 128, 1, None),
    (BF, 2, 40, 4, 2, 64, 128, 17, 5, [128, 60]),       # several row tiles
    (FP, 3, 3, 33, 1, 96, 90, 90, 0, [90, 64, 65]),     # 99 rows on one K/V head
    (BF, 2, 1, 4, 2, 16, 50, 0, 0, [-4, 1000]),         # lengths outside the cache are clamped
    (BF, 2, 3, 4, 2, 128, 200, 5, 200, [200, 66]),      # every key a sink
    (FP, 2, 2, 16, 2, 256, 640, 640, 0, [640, 577]),
    (BF, 2, 1, 6, 3, 32, 150, 150, 0, [150, 63]),
    (BF, 1, 2, 4, 1, 160, 400, 100, 8, [400]),
    (FP, 1, 2, 4, 1, 192, 400, 300, 8, [399]),
    (BF, 1, 1, 4, 1, 224, 400, 400, 0, [333]),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_decode(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, B, T, H, Hk, D, S, left, sinks, lens = case
    say("decode_q4", case)
    q = rand((B, T, H * D), 3, dtype, gpu)
    c = Q.cache(B, S, Hk, D, gpu, 4)
    if lens is None:
        lens = torch.randint(T, S + 1, (B,), generator=torch.Generator().manual_seed(3)).tolist()
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    o, lse = fta.flash_window_attn_decode_q4(q, c, ln, H, left, sinks, num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, Q.attend(q, c, lens, H, Hk, left, sinks, D ** -0.5), ("o", "lse"), str(case))


@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_unseen_rows_may_hold_anything(gpu, D):
    """Scales past the lengths, and between the sinks and the window, hold NaN and infinities."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, S, left, sinks, lens = 3, 2, 4, 2, 400, 50, 5, [399, 0, 207]
    q = rand((B, T, H * D), 3, BF, gpu)
    c = Q.cache(B, S, Hk, D, gpu, 4)
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    clean = fta.flash_window_attn_decode_q4(q, c, ln, H, left, sinks, num_kv_heads=Hk)
    for b in range(B):
        for x, bad in ((c.k_scales, math.nan), (c.v_scales, math.inf)):
            x[b, :, lens[b]:] = bad
            x[b, :, sinks:max(sinks, lens[b] - T - left)] = bad
    dirty = fta.flash_window_attn_decode_q4(q, c, ln, H, left, sinks, num_kv_heads=Hk)
    for x, y in zip(clean, dirty):
        assert torch.equal(x, y)
    assert (dirty[0][1] == 0).all() and (dirty[1][1] == -math.inf).all()


@pytest.mark.parametrize("dtype,scale", [(BF, 1e-3), (BF, 3e3), (FP, 1e-3), (FP, 300.0)])
def test_values_of_any_size(gpu, dtype, scale):
    """Values far from 1: scales times probabilities leave float16's normal range."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 2, 1, 8, 2, 128, 2000
    q = rand((B, T, H * D), 3, dtype, gpu)
    c = Q.cache(B, S, Hk, D, gpu, 4)
    c.v_scales.mul_(scale)
    ln = torch.tensor([S, 1500], dtype=torch.int32, device=gpu)
    o, lse = fta.flash_window_attn_decode_q4(q, c, ln, H, S, num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, Q.attend(q, c, ln.tolist(), H, Hk, S, 0, D ** -0.5), ("o", "lse"))


# interleaved pairs, tokens enough that a different order of the rotation's two products shows in 16 bits
INTERLEAVED = [
    (FP, 3, 386, 900, 3, 1, 16, 16, True, [121, 82, 342]),
    (FP, 1, 278, 250, 20, 4, 256, 16, True, [250]),
    (FP, 4, 150, 94, 11, 1, 224, 160, True, [13, 94, 94, 32]),
    (FP, 4, 97, 39, 64, 4, 96, 64, True, [22, 25, 39, 39]),
    (BF, 3, 217, 900, 8, 1, 112, 32, True, [174, 426, 541]),
    (BF, 2, 2000, 2000, 8, 2, 128, 128, True, [2000, 1999]),
]


@pytest.mark.parametrize("case", INTERLEAVED, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_append_of_interleaved_pairs(gpu, case):
    test_append(gpu, case)
