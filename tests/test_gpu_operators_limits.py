"""Calls of the operators around the sparse attention that are refused, or were once wrong, on the card."""

import math
import warnings

import pytest
import torch

from _helpers import rand

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


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


@pytest.mark.parametrize("dtype,H,Hk,D,Rc,inter", [(BF, 4, 2, 64, 64, False), (FP, 3, 1, 16, 16, True), (BF, 5, 5, 48, 32, False),
                                                   (FP, 2, 1, 128, 64, True), (BF, 2, 2, 256, 256, False)])
def test_padding_of_a_trained_layer_may_hold_anything(gpu, dtype, H, Hk, D, Rc, inter):
    """Preparation and window attention over a padded batch: what q, k and v hold behind seq_lens reaches no
    gradient, the norm weights' neither."""
    import flash_topk_attn_v2 as fta

    B, N, lens = 3, 70, [33, 0, 69]
    q, do = (rand((B, N, H * D), i, dtype, gpu) for i in (1, 2))
    k, v = (rand((B, N, Hk * D), i, dtype, gpu) for i in (3, 4))
    cos, sin = _tables(N, Rc, gpu)
    weights = [1 + 0.3 * rand((D,), i, torch.float32, gpu) for i in (5, 6)]
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)

    def grads():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, *weights)]
        a, b = fta.flash_qk_norm_rope(leaves[0], leaves[1], H, cos, sin, *leaves[3:], num_kv_heads=Hk, interleaved=inter)
        o, _ = fta.flash_window_attn(a, b, leaves[2], H, (20, 0), 3, num_kv_heads=Hk, seq_lens=ln)
        return torch.autograd.grad(o, leaves, do)

    clean = grads()
    for x, bad in zip((q, k, v, do), (math.nan, math.inf, -math.inf, math.nan)):
        for b in range(B):
            x[b, lens[b]:] = bad
    k[2, 69, ::3] = math.nan
    dirty = grads()
    for x, y in zip(clean, dirty):
        assert y.isfinite().all() and torch.equal(x, y)
    for x in dirty[:3]:
        for b in range(B):
            assert (x[b, lens[b]:] == 0).all()


def test_zero_gradients_in_some_rows_and_columns(gpu):
    """Heads with a zero gradient beside heads without, and gradients of a single column (of either sign of
    zero elsewhere): the same as one token at a time."""
    import flash_topk_attn_v2 as fta

    N, H, D = 8, 3, 64
    q, k = rand((1, N, H * D), 1, BF, gpu), rand((1, N, D), 2, BF, gpu)
    cos, sin = _tables(N, D, gpu)
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    dq[0, 0, :D], dq[0, 1, D + 7], dq[0, 2, 2 * D + 63] = rand((D,), 3, BF, gpu), 1.0, -2.0
    dq[0, 3], dk[0, 4, 0], dk[0, 5] = -0.0, 3.0, -0.0
    ql, kl = (x.clone().requires_grad_(True) for x in (q, k))
    got = torch.autograd.grad(fta.flash_qk_norm_rope(ql, kl, H, cos, sin, num_kv_heads=1), (ql, kl), (dq, dk))
    for x, d, g, heads in ((q, dq, got[0], H), (k, dk, got[1], 1)):
        live = (d.view(N, heads, D) != 0).any(-1)
        assert torch.equal((g.view(N, heads, D) != 0).any(-1), live)
    for n in range(N):
        a, b = (x[:, n:n + 1].clone().requires_grad_(True) for x in (q, k))
        pos = torch.tensor([n], dtype=torch.int32, device=gpu)
        one = torch.autograd.grad(fta.flash_qk_norm_rope(a, b, H, cos, sin, num_kv_heads=1, positions=pos), (a, b),
                                  (dq[:, n:n + 1], dk[:, n:n + 1]))
        assert torch.equal(one[0], got[0][:, n:n + 1]) and torch.equal(one[1], got[1][:, n:n + 1])


def test_append_warns_of_short_tables(gpu):
    """A cache that is longer than the tables: the tokens past them are turned as the last row, with a warning."""
    import flash_topk_attn_v2 as fta
    from flash_topk_attn_v2 import qk_prep

    H, D, S = 1, 64, 9
    q, k, v = (rand((1, 1, H * D), i, BF, gpu) for i in range(3))
    kc, vc = (torch.zeros(1, S, H * D, device=gpu, dtype=BF) for _ in range(2))
    lens = torch.tensor([S], dtype=torch.int32, device=gpu)
    cos, sin = _tables(S, D, gpu)
    qk_prep._warn_of_short_tables.cache_clear()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        full = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos, sin)
    with pytest.warns(UserWarning, match="nearest row"):
        short = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos[:S - 1], sin[:S - 1])
    last = fta.flash_qk_norm_rope(q, k, H, cos, sin, positions=torch.tensor([S - 2], dtype=torch.int32, device=gpu))[0]
    assert torch.equal(short, last) and not torch.equal(full, short)


def test_fractions_are_refused(gpu):
    import flash_topk_attn_v2 as fta

    x = torch.zeros(1, 5, 128, device=gpu, dtype=BF)
    cos, sin = _tables(5, 64, gpu)
    lens = torch.tensor([5], dtype=torch.int32, device=gpu)
    calls = [(fta.flash_window_attn, dict(q=x, k=x, v=x, num_heads=2, window=(3, 0), num_sinks=1, num_kv_heads=2),
              [dict(num_heads=2.5), dict(num_kv_heads=1.5), dict(window=(3.9, 0)), dict(window=(3, 0.1)), dict(num_sinks=0.5)]),
             (fta.flash_qk_norm_rope, dict(q=x, k=x, num_heads=2, cos=cos, sin=sin, num_kv_heads=2),
              [dict(num_heads=2.5), dict(num_kv_heads=2.5)]),
             (fta.flash_qk_norm_rope_append, dict(q=x, k=x, v=x, k_cache=x.clone(), v_cache=x.clone(), cache_lens=lens,
                                                  num_heads=2, cos=cos, sin=sin), [dict(num_heads=2.5), dict(position_offset=0.5)]),
             (fta.flash_window_attn_decode, dict(q=x, k_cache=x, v_cache=x, cache_lens=lens, num_heads=2, window_left=3),
              [dict(num_heads=2.5), dict(window_left=2.5), dict(num_sinks=1.5)]),
             (fta.flash_prefix_attn_decode, dict(q=x, k_prefix=x[0], v_prefix=x[0], k_cache=x, v_cache=x, cache_lens=lens,
                                                 num_heads=2), [dict(num_heads=2.5), dict(num_kv_heads=0.5)])]
    for call, good, bad in calls:
        call(**good)
        call(**(good | dict(num_heads=2.0)))
        for b in bad:
            with pytest.raises(ValueError, match="whole number"):
                call(**(good | b))
