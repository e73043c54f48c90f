"""Attention over 4-bit caches of as many new tokens as a prompt, or a part of one, has."""

import pytest
import torch

import _operators_ref as R
import _q4_ref as Q
import test_gpu_evict as E
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


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
def test_a_prompt_over_the_rows_read_back(gpu, dtype):
    """A prompt into a 4-bit cache, its attention over what the cache gives back in 16 bits, and the weights of the 4-bit
    keys by that attention's lse; a part of a prompt by the cache attention."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, left = 2, 300, 8, 2, 64, 120
    say("read back", dtype)
    q, k, v = (rand((B, T, h * D), 3 + i, dtype, gpu) for i, h in enumerate((H, Hk, Hk)))
    c = fta.flash_q4_cache(B, T, Hk, D, gpu)
    lens = torch.full((B,), T, dtype=torch.int32, device=gpu)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    q = fta.flash_qk_norm_rope_append_q4(q, k, v, c, lens, H, ang.cos().float().to(gpu), ang.sin().float().to(gpu), num_kv_heads=Hk)
    k16, v16 = fta.flash_q4_cache_read(c, D, dtype)
    o, lse = fta.flash_window_attn(q, k16, v16, H, (left, 0), num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, R.cache(q, k16, v16, [T] * B, H, Hk, left, 0, D ** -0.5), ("o", "lse"))
    part = torch.tensor([200, 300], dtype=torch.int32, device=gpu)
    got = fta.flash_window_attn_decode(q[:, 150:200], k16, v16, part, H, left, num_kv_heads=Hk)
    R.check(dict(zip(("o", "lse"), got)), R.cache(q[:, 150:200], k16, v16, part.tolist(), H, Hk, left, 0, D ** -0.5), ("o", "lse"))
    w = fta.flash_cache_weights(q, c, lse, lens, torch.zeros(B, Hk, T, device=gpu), H, left, num_kv_heads=Hk)
    keys = Q.values(c.k_codes, c.k_scales, True, D)[0]
    want, tol = E._weights(q, keys, lse, [T] * B, H, Hk, left, 0, D ** -0.5)
    assert ((w.double() - want).abs() <= tol + 2.0 ** -23 * w.double()).all()
