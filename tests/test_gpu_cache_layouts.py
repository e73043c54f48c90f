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


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_weights_that_overlap_what_is_read_are_refused(gpu, q4):
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 2, 4, 4, 2, 64, 48
    buf = torch.zeros(B * T * H * D * 2 + B * S * Hk * D * 2 + 64, dtype=torch.uint8, device=gpu)
    cache = Q.cache(B, S, Hk, D, gpu, 4) if q4 else rand((B, S, Hk * D), 4, BF, gpu)
    q = rand((B, T, H * D), 3, BF, gpu)
    ln = torch.tensor([40, 9], dtype=torch.int32, device=gpu)
    lse = torch.full((B, H, T), 3.0, device=gpu)
    want = fta.flash_cache_weights(q, cache, lse, ln, torch.zeros(B, Hk, S, device=gpu), H, S, num_kv_heads=Hk)
    n = 4 * B * Hk * S
    w = buf[:n].view(torch.float32).view(B, Hk, S)
    qs = buf[n - 16:][:B * T * H * D * 2].view(BF).view(B, T, H * D)
    ls = buf[n - 4:][:4 * B * H * T].view(torch.float32).view(B, H, T)
    li = buf[n // 2:][:4 * B].view(torch.int32)
    if q4:
        held = [cache._replace(v_scales=buf[n - 64:][:2 * cache.v_scales.numel()].view(FP).view_as(cache.v_scales)),
                cache._replace(k_codes=buf[:cache.k_codes.numel()].view_as(cache.k_codes))]
    else:
        held = [buf[n - 16:][:2 * cache.numel()].view(BF).view_as(cache)]
    for a in (dict(q=qs), dict(lse=ls), dict(cache_lens=li), *(dict(cache=x) for x in held)):
        with pytest.raises(ValueError, match="overlap"):
            fta.flash_cache_weights(**{**dict(q=q, cache=cache, lse=lse, cache_lens=ln, weights=w, num_heads=H, window_left=S, num_kv_heads=Hk), **a})
    assert not buf.any()
    # parts of one buffer that do not meet
    both = torch.zeros(B, 2, Hk, S, device=gpu)
    ls = both[:, 0].reshape(B, -1)[:, :H * T].view(B, H, T)
    ls.fill_(3.0)
    assert torch.equal(fta.flash_cache_weights(q, cache, ls, ln, both[:, 1], H, S, num_kv_heads=Hk), want)


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_requests_that_lie_between_each_other(gpu, q4):
    """Keys, values and weights of a request side by side in one buffer, requests behind each other; and an
    eviction into the caches of the requests between."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 3, 2, 4, 2, 64, 96
    lens = torch.tensor([96, 50, 7], dtype=torch.int32, device=gpu)
    n = 4 * Hk * S
    if q4:
        sizes = [32 * Hk * S, 4 * Hk * S] * 2 + [n]
        raw = torch.zeros(2 * B, sum(sizes), dtype=torch.uint8, device=gpu)
        codes, scales = (lambda x: x.view(2 * B, Hk, S, 32)), (lambda x: x.view(FP).view(2 * B, Hk, S, 2))
        views = (codes, scales, codes, scales)
    else:
        sizes = [2 * S * Hk * D] * 2 + [n]
        raw = torch.zeros(2 * B, sum(sizes), dtype=torch.uint8, device=gpu)
        views = (lambda x: x.view(BF).view(2 * B, S, Hk * D),) * 2
    at = [sum(sizes[:i]) for i in range(len(sizes))]
    parts = [f(raw[:, a:a + s]) for f, a, s in zip((*views, lambda x: x.view(torch.float32).view(2 * B, Hk, S)), at, sizes)]
    full = Q.cache(2 * B, S, Hk, D, gpu, 3) if q4 else tuple(rand((2 * B, S, Hk * D), 3 + i, BF, gpu) for i in (0, 1))
    for x, y in zip(parts, full):
        x.copy_(y)
    kind = (lambda t: fta.Q4Cache(*t)) if q4 else tuple
    mine, to = ((kind([t[i::2] for t in parts[:-1]]), parts[-1][i::2]) for i in (0, 1))
    own, own_to = ((kind([t.clone(memory_format=torch.contiguous_format) for t in c]), w.clone(memory_format=torch.contiguous_format))
                   for c, w in (mine, to))
    cos, sin = _tables(S, D // 2, gpu)
    q, k, v = (rand((B, T, h * D), i, BF, gpu) for i, h in enumerate((H, Hk, Hk)))
    for c, w in (mine, own):
        if q4:
            qr = fta.flash_qk_norm_rope_append_q4(q, k, v, c, lens, H, cos, sin, num_kv_heads=Hk)
            _, lse = fta.flash_window_attn_decode_q4(qr, c, lens, H, S, num_kv_heads=Hk)
        else:
            qr = fta.flash_qk_norm_rope_append(q, k, v, *c, lens, H, cos, sin, num_kv_heads=Hk)
            _, lse = fta.flash_window_attn_decode(qr, *c, lens, H, S, num_kv_heads=Hk)
        fta.flash_cache_weights(qr, c if q4 else c[0], lse, lens, w, H, S, num_kv_heads=Hk)
    got = fta.flash_cache_evict(*mine, lens, 40, 8, 2, out=to)
    want = fta.flash_cache_evict(*own, lens, 40, 8, 2, out=own_to)
    got2, want2 = (fta.flash_cache_evict(c, w, lens, 30, 8, 2) for c, w in (mine, own))
    for a, b in zip((*got, *got2, *mine[0], mine[1], *to[0], to[1]), (*want, *want2, *own[0], own[1], *own_to[0], own_to[1])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_an_eviction_reads_what_requests_and_heads_share(gpu, q4):
    """Into another cache: one prompt's cache for every request, one row of weights for every head."""
    import flash_topk_attn_v2 as fta

    B, Hk, D, S = 3, 2, 96, 150
    one = Q.cache(1, S, Hk, D, gpu, 3) if q4 else tuple(rand((1, S, Hk * D), 3 + i, BF, gpu) for i in (0, 1))
    w = torch.rand(B, 1, S, device=gpu).expand(B, Hk, S)
    lens = torch.tensor([150, 99, 20], dtype=torch.int32, device=gpu)
    kind = (lambda t: fta.Q4Cache(*t)) if q4 else tuple
    shared = kind([t.expand(B, *t.shape[1:]) for t in one])
    done = []
    for c, x in ((shared, w), (kind([t.contiguous() for t in shared]), w.contiguous())):
        to = Q.cache(B, 70, Hk, D, gpu, 5) if q4 else tuple(rand((B, 70, Hk * D), 7 + i, BF, gpu) for i in (0, 1))
        to = to, torch.ones(B, Hk, 70, device=gpu)
        done.append((*fta.flash_cache_evict(c, x, lens, 60, 8, 2, out=to), *to[0], to[1]))
    for a, b in zip(*done):
        assert torch.equal(a, b)
    for bad in (dict(cache=shared, weights=w.contiguous()), dict(cache=kind([t.contiguous() for t in shared]), weights=w)):
        with pytest.raises(ValueError, match="share memory"):
            fta.flash_cache_evict(**bad, cache_lens=lens, budget=60)


@pytest.mark.parametrize("out", [False, True], ids=["in_place", "out"])
def test_an_eviction_whose_weights_hold_the_lengths_is_refused(gpu, out):
    """The lengths are read while weights are written."""
    import flash_topk_attn_v2 as fta

    B, Hk, D, S = 2, 2, 64, 40
    cache, other = (tuple(rand((B, S, Hk * D), 2 * i + j, BF, gpu) for j in (0, 1)) for i in (0, 1))
    w, free = torch.rand(B, Hk, S, device=gpu), torch.rand(B, Hk, S, device=gpu)
    held = [x.clone() for x in (*cache, w)]
    lens = w.view(torch.int32)[1, 1, 5:5 + B]
    with pytest.raises(ValueError, match="overlap"):
        fta.flash_cache_evict(cache, free if out else w, lens, 10, out=(other, w) if out else None)
    assert all(torch.equal(x, y) for x, y in zip(held, (*cache, w)))
    # lengths between the rows of weights
    wide = torch.zeros(B, Hk, S + 8, device=gpu)
    lens = wide.view(torch.int32)[0, 0, S:S + B]
    lens.copy_(torch.tensor([40, 33], dtype=torch.int32))
    part = wide[:, :, :S]
    part.copy_(w)
    got = fta.flash_cache_evict(cache, part, lens, 10)
    want = fta.flash_cache_evict(tuple(x.clone() for x in held[:2]), w, torch.tensor([40, 33], dtype=torch.int32, device=gpu), 10)
    assert torch.equal(got[1], want[1]) and torch.equal(part, w) and lens.tolist() == [40, 33]
