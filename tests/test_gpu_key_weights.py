"""Key weights by the kernel that takes them: rows in registers ("step"), rows held in LDS ("held"), rows that
come through LDS in chunks ("many")."""

import math

import pytest
import torch

import _q4_ref as Q
import test_gpu_evict as E
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def path(T, G):
    """``(kernel, heads GG, tokens TT of a chunk of 32 rows)`` of T tokens, G query heads on a K/V head."""
    gg = min(G, max(1, 32 // min(T, 32)))
    tt = 32 // gg
    chunks = -(-T // tt) * -(-G // gg)
    return "step" if T * G <= 32 else "held" if chunks <= 4 else "many", gg, tt


# T, H, Hk, D, left, sinks; the kernel, and the rows of a chunk that hold a token's head
NOT_FINITE = [
    (8, 3, 1, 64, 5, 0, "step", None),
    (5, 12, 2, 128, 11, 2, "step", None),
    (9, 8, 2, 64, 5, 0, "held", 30),
    (5, 16, 2, 128, 40, 3, "held", 30),
    (64, 4, 2, 64, 7, 0, "held", 32),
    (9, 26, 2, 64, 7, 0, "many", 30),
    (70, 5, 5, 64, 9, 0, "held", 32),
    (10, 33, 1, 128, 200, 0, "many", 30),
    (140, 5, 5, 64, 9, 1, "many", 32),
    (190, 6, 2, 256, 200, 0, "many", 32),
    (900, 8, 2, 64, 960, 0, "many", 32),    # walks in several parts
    (500, 20, 4, 128, 300, 9, "many", 32),
]


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case", NOT_FINITE, ids=lambda c: "-".join(str(x) for x in c))
def test_a_token_without_a_finite_lse_stays_with_its_keys(gpu, case, q4):
    """A query of NaN makes its lse NaN, as the attention gives it: the keys that its token sees have no finite sum
    then, the others keep every bit."""
    import flash_topk_attn_v2 as fta

    T, H, Hk, D, left, sinks, kernel, rows = case
    say("not finite", case, q4)
    got = path(T, H // Hk)
    assert got[0] == kernel and rows in (None, got[1] * got[2])
    n = 200 if T < 200 else T + 60
    S = n + 40
    q = rand((1, T, H * D), 3, BF, gpu)
    cache = Q.cache(1, S, Hk, D, gpu, 4) if q4 else rand((1, S, Hk * D), 4, BF, gpu)
    ln = torch.tensor([n], dtype=torch.int32, device=gpu)

    def weigh(q):
        if q4:
            _, lse = fta.flash_window_attn_decode_q4(q, cache, ln, H, left, sinks, num_kv_heads=Hk)
        else:
            _, lse = fta.flash_window_attn_decode(q, cache, cache, ln, H, left, sinks, num_kv_heads=Hk)
        zero = torch.zeros(1, Hk, S, device=gpu)
        return lse, fta.flash_cache_weights(q, cache, lse, ln, zero, H, left, sinks, num_kv_heads=Hk)

    _, want = weigh(q)
    assert want.isfinite().all()
    for t in sorted({0, 1, T // 2, T - 1}):
        bad = q.clone()
        bad[:, t] = math.nan
        lse, w = weigh(bad)
        assert lse[:, :, t].isnan().all() and lse.isnan().sum() == H
        p = n - T + t
        sees = torch.zeros(S, dtype=torch.bool, device=gpu)
        sees[max(0, p - left):p + 1] = True
        sees[:min(sinks, p + 1)] = True
        assert w[0, :, sees].isnan().all(), t
        assert torch.equal(w[0, :, ~sees], want[0, :, ~sees]), t


# dtype, B, T, H, Hk, D, S, left, sinks, lens; the kernel and the rows of a chunk that are used
BY_KERNEL = [
    ((BF, 2, 9, 26, 2, 128, 300, 120, 3, [300, 77]), "many", 30),      # 13 heads of a K/V head, three at a time
    ((FP, 1, 10, 33, 1, 64, 500, 500, 0, [499]), "many", 30),
    ((BF, 2, 6, 28, 2, 64, 260, 100, 2, [260, 5]), "held", 30),          # 14 heads, five at a time: the last one is short
    ((FP, 2, 9, 8, 2, 80, 700, 300, 0, [700, 8]), "held", 30),          # four heads, three at a time
    ((BF, 3, 12, 20, 4, 128, 900, 900, 0, [900, 300, 12]), "held", 32),
    ((BF, 2, 12, 40, 4, 80, 2100, 300, 100, [2099, 40]), "many", 32),   # ten heads, two at a time: five chunks
    ((FP, 3, 33, 6, 2, 64, 1200, 1200, 3, [1200, 33, 1]), "many", 32),  # two chunks a head, the second of one token
    ((BF, 1, 20, 10, 2, 128, 640, 640, 0, [640]), "many", 32),
    ((FP, 2, 4, 8, 2, 192, 700, 500, 3, [700, 129]), "step", None),
    ((BF, 2, 5, 12, 2, 192, 700, 500, 3, [700, 129]), "step", None),     # 30 rows: two tiles of 16
    ((BF, 2, 8, 8, 2, 224, 700, 700, 0, [690, 3]), "step", None),
    ((FP, 1, 1, 8, 2, 224, 700, 700, 0, [700]), "step", None),
    ((FP, 2, 8, 8, 2, 256, 400, 400, 0, [400, 65]), "step", None),
    ((BF, 2, 8, 8, 2, 128, 400, 400, 0, [400, 65]), "step", None),
    ((BF, 2, 16, 8, 2, 192, 600, 600, 0, [600, 20]), "held", 32),
    ((FP, 2, 16, 8, 2, 224, 600, 130, 5, [600, 20]), "held", 32),
    ((FP, 1, 64, 4, 2, 256, 700, 700, 0, [700]), "held", 32),
    ((BF, 1, 100, 8, 2, 192, 400, 400, 0, [400]), "many", 32),
    ((FP, 1, 100, 8, 2, 224, 400, 90, 7, [333]), "many", 32),
    ((FP, 1, 300, 8, 2, 256, 400, 400, 0, [399]), "many", 32),
    ((BF, 2, 100, 8, 2, 32, 400, 400, 0, [400, 99]), "many", 32),
]


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
@pytest.mark.parametrize("case,kernel,rows", BY_KERNEL, ids=lambda c: "-".join(str(x) for x in c[1:9]) if isinstance(c, tuple) else str(c))
def test_weights_by_kernel(gpu, case, kernel, rows, q4):
    got = path(case[2], case[3] // case[4])
    assert got[0] == kernel and rows in (None, got[1] * got[2])
    E.test_weights(gpu, case, q4)


# caches whose selection holds 32 weights a thread, and the ends of that range: B, Hk, D, S, budget, recent, sinks, lens
SELECT = [
    (1, 2, 32, 20000, 3000, 100, 4, [19999]),
    (2, 1, 16, 32768, 20000, 0, 0, [32768, 20001]),
    (1, 1, 32, 16385, 1, 0, 0, [16385]),
    (1, 1, 16, 32769, 5000, 64, 4, [32769]),
    (1, 1, 16, 16384, 16383, 5, 5, [16384]),
]


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "out"])
@pytest.mark.parametrize("case", SELECT, ids=lambda c: "-".join(str(x) for x in c[:7]))
def test_selection_of_long_heads(gpu, case, out):
    E.test_evict(gpu, case, True, out)
