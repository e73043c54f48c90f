"""Calls of the operators around the sparse attention that are refused, or were once wrong, on the card."""

import pytest
import torch

from _helpers import rand

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _tables(P, Rc, dev):
    inv = 10000.0 ** (-torch.arange(0, Rc, 2, dtype=torch.float64) / Rc)
    a = torch.arange(P, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(dev), a.sin().float().to(dev)


def test_append_refuses_caches_that_share_memory(gpu):
    """K and V written to the same rows would leave whichever is stored last."""
    import flash_topk_attn_v2 as fta

    B, T, H, D, S = 2, 1, 2, 64, 9
    q, k, v = (rand((B, T, H * D), i, BF, gpu) for i in range(3))
    cos, sin = _tables(S, D, gpu)
    lens = torch.tensor([3, 9], dtype=torch.int32, device=gpu)
    both = torch.zeros(B, S, 3 * H * D, device=gpu, dtype=BF)
    one, two, three = both.split(H * D, -1)
    fta.flash_qk_norm_rope_append(q, k, v, one, three, lens, H, cos, sin)
    before = both.clone()
    half = both[..., 64:64 + H * D]
    for kc, vc in ((one, one), (one, half), (half, two), (both.view(-1).as_strided((B, S, H * D), (64, H * D, 1)), three)):
        with pytest.raises(ValueError, match="share memory"):
            fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos, sin)
    assert torch.equal(both, before)
