"""Key weights by the kernel that takes them: rows in registers ("step"), rows held in LDS ("held"), rows that
come through LDS in chunks ("many")."""

import math

import pytest
import torch

import _q4_ref as Q
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
