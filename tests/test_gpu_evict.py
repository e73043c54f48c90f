"""The attention that cached keys receive, and the eviction by it, against their definitions."""

import math

import pytest
import torch

import _operators_ref as R
import _q4_ref as Q
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _weights(q, keys, lse, lens, H, Hk, left, sinks, scale):
    """``flash_cache_weights`` of keys [B, Hk, S, D] in float64.

    Every term is off by at most F4 of it (the exponent's fp32 arithmetic; 4-bit keys the more of the
    two kinds) and by the lse's own rounding; sums of n positive terms by n 2^-24 of the sum at most,
    here in chunks of 32 rows, runs of 64 chunks and their sum.
    """
    B, T, C = q.shape
    D, G, S, dev = C // H, H // Hk, keys.shape[2], q.device
    w, tol = (torch.zeros(B, Hk, S, device=dev, dtype=torch.float64) for _ in range(2))
    for b in range(B):
        n = max(0, min(S, int(lens[b])))
        if n == 0:
            continue
        see = R.window_mask(T, n, n - T, left, 0, sinks, dev)
        for h in range(H):
            s = (q[b].view(T, H, D)[:, h].double() @ keys[b, h // G, :n].T * scale).masked_fill(~see, -math.inf)
            x = torch.exp(s - lse[b, h, :, None].double().masked_fill(lse[b, h, :, None] == -math.inf, math.inf))
            w[b, h // G, :n] += x.sum(0)
            tol[b, h // G, :n] += (x * (Q.F4 + 2.0 ** -22 * lse[b, h, :, None].double().abs().nan_to_num(posinf=0))).sum(0)
    sums = (32 + 64 + T * G / 2048 + 16) * 2.0 ** -24
    return w, tol + sums * w + T * G * R.FLUSH


# dtype, B, T, H, Hk, D, S, left, sinks, lens
WEIGHTS = [
    (BF, 1, 1, 1, 1, 64, 1, 0, 0, [1]),
    (BF, 4, 1, 8, 2, 128, 300, 20, 4, [300, 1, 0, 157]),
    (FP, 3, 2, 4, 4, 64, 333, 100, 0, [333, 200, 64]),
    (BF, 2, 1, 8, 1, 256, 700, 10000, 3, [700, 129]),
    (FP, 2, 5, 16, 2, 80, 300, 31, 33, [3, 300]),       # fewer tokens than new ones
    (BF, 1, 3, 12, 2, 128, 260, 255, 0, [259]),         # groups of six heads: 30 rows of 32
    (FP, 2, 7, 33, 1, 96, 200, 200, 0, [200, 64]),      # 33 heads on one K/V head
    (BF, 2, 100, 4, 2, 64, 100, 100, 0, [100, 60]),     # a prompt, padded batch
    (BF, 1, 700, 8, 2, 128, 700, 700, 0, [700]),        # parts
    (FP, 1, 700, 6, 2, 64, 700, 99, 10, [700]),         # with a window and sinks
    (BF, 2, 33, 4, 4, 256, 500, 500, 0, [500, 40]),
    (BF, 2, 1, 4, 2, 16, 50, 0, 0, [-4, 1000]),
    (BF, 1, 20, 40, 1, 48, 129, 60, 2, [129]),
    (FP, 1, 40, 4, 4, 160, 140, 140, 0, [140]),
]


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case", WEIGHTS, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_weights(gpu, case, q4):
    import flash_topk_attn_v2 as fta

    dtype, B, T, H, Hk, D, S, left, sinks, lens = case
    say("weights", case, q4)
    q = rand((B, T, H * D), 3, dtype, gpu)
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    if q4:
        cache = Q.cache(B, S, Hk, D, gpu, 4)
        keys = Q.values(cache.k_codes, cache.k_scales, True, D)[0]
        _, lse = fta.flash_window_attn_decode_q4(q, cache, ln, H, left, sinks, num_kv_heads=Hk)
    else:
        cache = rand((B, S, Hk * D), 4, dtype, gpu)
        keys = cache.view(B, S, Hk, D).transpose(1, 2).double()
        _, lse = fta.flash_window_attn_decode(q, cache, cache, ln, H, left, sinks, num_kv_heads=Hk)
    start = torch.rand(B, Hk, S, generator=torch.Generator().manual_seed(1)).to(gpu)
    w = start.clone()
    assert fta.flash_cache_weights(q, cache, lse, ln, w, H, left, sinks, num_kv_heads=Hk) is w
    want, tol = _weights(q, keys, lse, lens, H, Hk, left, sinks, D ** -0.5)
    assert ((w.double() - start.double() - want).abs() <= tol + 2.0 ** -23 * (w.double() + start.double())).all()
    for b in range(B):  # rows behind the length
        assert torch.equal(w[b, :, max(0, lens[b]):], start[b, :, max(0, lens[b]):])
    # every token that sees something gives 1 per head, in all
    live = (lse > -math.inf).sum((1, 2)).double()
    assert ((want.sum((1, 2)) - live).abs() <= 1e-3 * live + 1e-12).all()


def _evicted(w, n, budget, recent, sinks):
    """Rows of one head that stay."""
    if n <= budget:
        return list(range(n))
    val = [(math.isnan(x), 0.0 if math.isnan(x) else -x) for x in w.tolist()]  # NaN last
    best = sorted(range(sinks, n - recent), key=lambda j: (val[j], j))[:budget - sinks - recent]
    return sorted([*range(sinks), *best, *range(n - recent, n)])


# B, Hk, D, S, budget, recent, sinks, lens
EVICT = [
    (1, 1, 64, 1, 1, 0, 0, [1]),
    (2, 2, 64, 40, 10, 3, 2, [40, 9]),
    (3, 2, 128, 300, 100, 0, 0, [300, 101, 0]),
    (2, 3, 80, 257, 64, 64, 0, [257, 64]),              # recent rows alone
    (2, 1, 16, 257, 64, 0, 64, [200, 65]),              # sinks alone
    (1, 2, 256, 1030, 1029, 17, 4, [1030]),             # one row goes
    (2, 2, 96, 700, 600, 30, 4, [5000, -3]),            # lengths outside the cache
    (1, 2, 64, 9000, 2000, 100, 4, [8999]),             # more rows than a thread's eight
    (1, 1, 32, 40000, 777, 10, 1, [39000]),             # more than its 32
    (20, 8, 128, 500, 123, 20, 4, None),
]


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "out"])
@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_evict(gpu, case, q4, out):
    import flash_topk_attn_v2 as fta

    B, Hk, D, S, budget, recent, sinks, lens = case
    say("evict", case, q4, out)
    gen = torch.Generator().manual_seed(7)
    if lens is None:
        lens = torch.randint(0, S + 1, (B,), generator=gen).tolist()
    w = torch.randn(B, Hk, S, generator=gen).exp()
    w = torch.where(torch.rand(B, Hk, S, generator=gen) < 0.4, (w * 4).round() / 4, w)  # ties
    w[torch.rand(B, Hk, S, generator=gen) < 0.1] = 0.0
    w[:, 0, S // 3:S // 2] = 0.25                                                    # a run of equal ones
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    if q4:
        cache = Q.cache(B, S, Hk, D, gpu, 4)
        rows = list(cache)
    else:
        cache = tuple(rand((B, S, Hk * D), 5 + i, BF, gpu) for i in (0, 1))
        rows = [x.view(B, S, Hk, D).transpose(1, 2) for x in cache]
    old = [x.clone() for x in rows]
    wg = w.to(gpu)
    to, to_rows, room = None, rows, S
    if out:
        room = budget + 5
        if q4:
            to = Q.cache(B, room, Hk, D, gpu, 9)
            to_rows = list(to)
        else:
            to = tuple(rand((B, room, Hk * D), 9 + i, BF, gpu) for i in (0, 1))
            to_rows = [x.view(B, room, Hk, D).transpose(1, 2) for x in to]
        to = (to, torch.ones(B, Hk, room, device=gpu))
    before = [x.clone() for x in to_rows]
    new, kept = fta.flash_cache_evict(cache, wg, ln, budget, recent, sinks, out=to)
    got_w = wg if to is None else to[1]
    assert new.dtype == kept.dtype == torch.int32 and kept.shape == (B, Hk, budget)
    for b in range(B):
        n = max(0, min(S, lens[b]))
        assert int(new[b]) == min(n, budget)
        for h in range(Hk):
            stay = _evicted(w[b, h], n, budget, recent, sinks)
            m = len(stay)
            assert kept[b, h, :m].tolist() == stay and (kept[b, h, m:] == -1).all()
            at = torch.tensor(stay, dtype=torch.long, device=gpu)
            for x, o, f in zip(to_rows, old, before):
                assert torch.equal(x[b, h, :m], o[b, h, at]) and torch.equal(x[b, h, m:], f[b, h, m:])
            want = w[b, h].to(gpu).clone() if to is None else torch.zeros(room, device=gpu)
            if to is None:
                want[m:n] = 0
            want[:m] = w[b, h].to(gpu)[at]
            assert torch.equal(got_w[b, h], want)
    if out:  # the inputs are as they were
        assert torch.equal(wg.cpu(), w) and all(torch.equal(x, o) for x, o in zip(rows, old))


def test_evict_of_special_weights(gpu):
    """NaN below everything, infinities, zeros of both signs, negative and subnormal numbers."""
    import flash_topk_attn_v2 as fta

    vals = [0.0, -0.0, math.nan, math.inf, -math.inf, -1.0, 1e-40, -1e-40, 1.0, 3.0e38, -math.nan, 2.0 ** -149]
    S = 4 * len(vals)
    w = torch.tensor(vals * 4)[None, None]
    cache = tuple(rand((1, S, 16), i, BF, gpu) for i in (0, 1))
    for budget in range(1, S, 5):
        c = tuple(x.clone() for x in cache)
        _, kept = fta.flash_cache_evict(c, w.to(gpu), torch.tensor([S], dtype=torch.int32, device=gpu), budget)
        assert kept[0, 0].tolist() == _evicted(w[0, 0], S, budget, 0, 0)


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("T,H,Hk,left,sinks", [(8, 3, 1, 5, 0), (64, 3, 1, 5, 0), (64, 12, 2, 40, 3), (70, 5, 5, 9, 0), (45, 33, 1, 7, 0)])
def test_a_token_that_is_not_finite_stays_with_its_keys(gpu, T, H, Hk, left, sinks, q4):
    """A query of NaN reaches the keys that its token sees and no others, whose sums keep every bit."""
    import flash_topk_attn_v2 as fta

    S, D = 200, 64
    q = rand((1, T, H * D), 3, BF, gpu)
    cache = Q.cache(1, S, Hk, D, gpu, 4) if q4 else rand((1, S, Hk * D), 4, BF, gpu)
    ln = torch.tensor([S - 9], dtype=torch.int32, device=gpu)
    lse = torch.full((1, H, T), 3.0, device=gpu)
    zero = torch.zeros(1, Hk, S, device=gpu)
    want = fta.flash_cache_weights(q, cache, lse, ln, zero.clone(), H, left, sinks, num_kv_heads=Hk)
    for t in (0, T // 2, T - 1):
        bad = q.clone()
        bad[:, t] = math.nan
        got = fta.flash_cache_weights(bad, cache, lse, ln, zero.clone(), H, left, sinks, num_kv_heads=Hk)
        p = S - 9 - T + t
        sees = torch.zeros(S, dtype=torch.bool, device=gpu)
        sees[max(0, p - left):p + 1] = True
        sees[:sinks] = True
        assert got[0, :, sees].isnan().all() and torch.equal(got[0, :, ~sees], want[0, :, ~sees])


# rows that stay in LDS while keys stream past: windows, sinks, lengths under T, several tiles of a wave
HELD = [
    (BF, 5, 24, 8, 2, 128, 3001, 1500, 40, [3001, 2000, 24, 10, 0]),
    (FP, 2, 128, 2, 2, 64, 5000, 5000, 0, [5000, 127]),
    (BF, 1, 12, 40, 4, 80, 2100, 300, 100, [2099]),          # ten heads: 30 rows of 32
    (FP, 3, 33, 6, 2, 256, 1200, 1200, 3, [1200, 33, 1]),
    (BF, 40, 9, 8, 2, 96, 4000, 2000, 0, None),
    (FP, 1, 64, 4, 2, 16, 70, 5, 1, [70]),
]


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case", HELD, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_weights_of_held_rows(gpu, case, q4):
    if case[-1] is None:
        case = (*case[:-1], torch.randint(0, case[6] + 1, (case[1],), generator=torch.Generator().manual_seed(2)).tolist())
    test_weights(gpu, case, q4)


# caches of more than 1024 rows (a workgroup selects, not a wave), and few rows of many heads (fewer threads move them)
EVICT_LONG = [
    (2, 3, 80, 1300, 64, 64, 0, [1300, 64]),
    (2, 1, 16, 1100, 64, 0, 64, [1100, 65]),
    (2, 2, 96, 2100, 600, 30, 4, [5000, -3]),
    (3, 2, 128, 1025, 1024, 0, 0, [1025, 1024, 7]),
    (1, 1, 64, 1024, 1000, 3, 1, [1024]),
    (64, 8, 64, 1100, 1000, 20, 4, None),
]


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "out"])
@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case", EVICT_LONG, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_evict_of_long_caches(gpu, case, q4, out):
    test_evict(gpu, case, q4, out)


@pytest.mark.parametrize("S", [1024, 1100])
def test_evict_of_special_weights_in_long_caches(gpu, S):
    import flash_topk_attn_v2 as fta

    vals = [0.0, -0.0, math.nan, math.inf, -math.inf, -1.0, 1e-40, -1e-40, 1.0, 3.0e38, -math.nan, 2.0 ** -149]
    w = torch.tensor(vals * (S // len(vals) + 1))[None, None, :S].contiguous()
    cache = tuple(rand((1, S, 16), i, BF, gpu) for i in (0, 1))
    for budget in range(1, S, 85):
        c = tuple(x.clone() for x in cache)
        _, kept = fta.flash_cache_evict(c, w.to(gpu), torch.tensor([S], dtype=torch.int32, device=gpu), budget)
        assert kept[0, 0].tolist() == _evicted(w[0, 0], S, budget, 0, 0)


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_out_that_is_the_input_is_refused_every_time(gpu, q4):
    """Also behind calls in place and into another cache of the same layout."""
    import flash_topk_attn_v2 as fta

    cache, other = (Q.cache(1, 40, 2, 64, gpu, 4 + i) if q4 else tuple(rand((1, 40, 128), 2 * i + j, BF, gpu) for j in (0, 1)) for i in (0, 1))
    w, w2 = (torch.rand(1, 2, 40, device=gpu) for _ in range(2))
    ln = torch.tensor([40], dtype=torch.int32, device=gpu)
    for _ in range(2):
        fta.flash_cache_evict(cache, w, ln, 10)
        fta.flash_cache_evict(cache, w, ln, 10, out=(other, w2))
        for out in ((cache, w), (cache, w2), (other, w)):
            with pytest.raises(ValueError, match="overlap"):
                fta.flash_cache_evict(cache, w, ln, 10, out=out)
