"""The calls over 4-bit and 16-bit caches on parts of larger ones, against the same on tensors of their own."""

import pytest
import torch

import _q4_ref as Q
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _tables(P, R2, dev):
    a = torch.arange(P, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(R2, dtype=torch.float64) / R2)
    return a.cos().float().to(dev), a.sin().float().to(dev)


@pytest.mark.parametrize("T", [1, 30, 180])
@pytest.mark.parametrize("D", [16, 96, 160, 224])
def test_scales_of_one_request(gpu, D, T):
    """One request of a contiguous cache of two whose heads have an odd number of scales: they start between two
    32-bit words."""
    import flash_topk_attn_v2 as fta

    H, Hk, S = 4, 1, 187
    say("one request", D, T)
    big = Q.cache(2, S, Hk, D, gpu, 3)
    c = fta.Q4Cache(*(t[1:] for t in big))
    own = fta.Q4Cache(*(t.clone() for t in c))
    other = [t[0].clone() for t in big]
    assert c.k_scales.data_ptr() % 4 == 2
    q, k, v = (rand((1, T, h * D), i, FP, gpu) for i, h in enumerate((H, Hk, Hk)))
    cos, sin = _tables(S, 8, gpu)
    ln = torch.tensor([S - 3], dtype=torch.int32, device=gpu)
    done = []
    for x in (c, own):
        qr = fta.flash_qk_norm_rope_append_q4(q, k, v, x, ln, H, cos, sin, num_kv_heads=Hk)
        o, lse = fta.flash_window_attn_decode_q4(qr, x, ln, H, 90, 4, num_kv_heads=Hk)
        w = torch.zeros(1, Hk, S, device=gpu)
        fta.flash_cache_weights(qr, x, lse, ln, w, H, 90, 4, num_kv_heads=Hk)
        to = Q.cache(2, 51, Hk, D, gpu, 5)
        out = fta.Q4Cache(*(t[1:] for t in to)), torch.ones(1, Hk, 51, device=gpu)
        new, kept = fta.flash_cache_evict(x, w, ln, 40, 8, 2, out=out)
        new2, kept2 = fta.flash_cache_evict(x, w, ln, 60, 8, 2)
        done.append((qr, o, lse, w, *to, out[1], new, kept, new2, kept2, *x, *fta.flash_q4_cache_read(x, D, BF)))
    for a, b in zip(*done):
        assert torch.equal(a, b)
    assert all(torch.equal(t[0], x) for t, x in zip(big, other))
