"""Attention over 4-bit caches of as many new tokens as a prompt, or a part of one, has."""

import pytest
import torch

import _operators_ref as R
import _q4_ref as Q
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16

# dtype, B, T, H, Hk, D, S, left, sinks, lens
PROMPTS = [
    (BF, 1, 2048, 4, 1, 128, 2048, 2048, 0, [2048]),
    (FP, 1, 2048, 2, 2, 64, 2100, 500, 5, [2077]),
    (BF, 2, 513, 6, 2, 96, 4000, 4000, 0, [4000, 300]),   # a part of a prompt; fewer tokens than new ones
    (FP, 1, 300, 8, 1, 256, 1500, 700, 9, [1500]),
    (BF, 3, 129, 12, 4, 80, 1000, 64, 0, [1000, 129, 128]),
]


@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_prompts(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, B, T, H, Hk, D, S, left, sinks, lens = case
    say("q4 prompt", case)
    q = rand((B, T, H * D), 3, dtype, gpu)
    c = Q.cache(B, S, Hk, D, gpu, 4)
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    o, lse = fta.flash_window_attn_decode_q4(q, c, ln, H, left, sinks, num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, Q.attend(q, c, lens, H, Hk, left, sinks, D ** -0.5), ("o", "lse"), str(case))


def test_a_prompt_in_parts(gpu):
    """A prompt of four parts: what each part's tokens see is what they see of the whole."""
    import flash_topk_attn_v2 as fta

    H, Hk, D, N, P = 8, 2, 64, 1000, 250
    q = rand((1, N, H * D), 3, BF, gpu)
    c = Q.cache(1, N, Hk, D, gpu, 4)
    ref = Q.attend(q, c, [N], H, Hk, N, 0, D ** -0.5)
    for t in range(0, N, P):
        ln = torch.tensor([t + P], dtype=torch.int32, device=gpu)
        o, lse = fta.flash_window_attn_decode_q4(q[:, t:t + P], c, ln, H, N, num_kv_heads=Hk)
        part = {n: (x[..., t:t + P] if n.startswith("lse") else x[:, t:t + P]) for n, x in ref.items()}
        R.check({"o": o, "lse": lse}, part, ("o", "lse"), f"part {t}")
