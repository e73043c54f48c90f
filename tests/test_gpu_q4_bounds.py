"""How far what a 4-bit cache holds is from what was appended, at every magnitude: the bound that the append documents."""

import pytest
import torch

import _q4_ref as Q
from _helpers import say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, FP], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 80, 128])
def test_columns_are_near_what_was_appended(gpu, D, dtype):
    """With t the largest magnitude over 8 and d the scale, |d| is off t by 2^-11 of t where it is a normal float16 and by
    2^-25 where it is not.  x / d is then at most 8 (1 + 2^-11) (to first order; 8 + 2^-8, with room for the second 8.004),
    or 8 + 2^-22 / |d|: the code nearest to it is off by half a scale, by what passes 8 at the end of code 0, by one more scale
    at the end of code 15.  Scales of 0 hold nothing: their groups' magnitudes are 2^-22 at most."""
    import flash_topk_attn_v2 as fta

    say("bounds", D, dtype)
    gen = torch.Generator().manual_seed(1)
    T, low = 4000, -30 if dtype == BF else -24
    mag = 2.0 ** (low + (18 - low if dtype == BF else 15 - low) * torch.rand(T, -(-D // 32), 1, generator=gen, dtype=torch.float64))
    x = mag * (2 * torch.rand(T, mag.shape[1], 32, generator=gen, dtype=torch.float64) - 1)
    x[::3, :, 5] = mag[::3, :, 0]
    x[::3, :, 9] = -mag[::3, :, 0] * (1 - 2.0 ** -6)
    v = x.flatten(-2)[:, :D].to(dtype).to(gpu)[None].contiguous()
    c = fta.flash_q4_cache(1, T, 1, D, gpu)
    tab = torch.zeros(T, 8, device=gpu)
    fta.flash_qk_norm_rope_append_q4(v, v, v, c, torch.tensor([T], dtype=torch.int32, device=gpu), 1, tab, tab)
    got, d = (t[0, 0] for t in Q.values(c.v_codes, c.v_scales, False, D))
    v = v[0].double()
    off = (got - v).abs()
    top = torch.nn.functional.pad(v, (0, -D % 32)).unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2)[:, :D]
    assert (top <= 8 * 65504).all()
    small = top < 2.0 ** -11
    first = torch.nn.functional.pad(v, (0, -D % 32)).unflatten(-1, (-1, 32))
    sign = torch.where(-first.amin(-1) >= first.amax(-1), -1.0, 1.0)[..., None].expand(-1, -1, 32).flatten(-2)[:, :D]
    opposite = sign * v < -7.5 * d + 2.0 ** -22 * small  # it is held to code 15
    bound = torch.where(opposite, d * (1 + 2.0 ** -8 + 2.0 ** -18), d / 2) + 2.0 ** -22 * small
    assert (off <= bound).all()
    assert (got[d == 0] == 0).all() and (top[d == 0] <= 2.0 ** -22).all()
    assert bool((off[small] > d[small]).any())  # where half a scale, or one, is not the bound
