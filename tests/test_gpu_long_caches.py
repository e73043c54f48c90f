"""4-bit caches, key weights and eviction as they are used together: steps of a serving batch,
captured graphs, other streams, views, long caches, and what is refused."""

import math

import pytest
import torch

import _operators_ref as R
import _q4_ref as Q
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _tables(P, R2, dev):
    a = torch.arange(P, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(R2, dtype=torch.float64) / R2)
    return a.cos().float().to(dev), a.sin().float().to(dev)


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_a_serving_batch(gpu, q4):
    """Prompts into the caches, steps that add up weights, an eviction, more steps: every output against
    a float64 model that keeps what the caches hold."""
    import flash_topk_attn_v2 as fta

    B, H, Hk, D, S, budget = 3, 8, 2, 64, 150, 70
    prompts, dtype = [100, 37, 64], BF
    cos, sin = _tables(400, D // 2, gpu)
    qw, kw = (1 + 0.1 * rand((D,), 8 + i, torch.float32, gpu) for i in (0, 1))
    weights = torch.zeros(B, Hk, S, device=gpu)
    if q4:
        cache = fta.flash_q4_cache(B, S, Hk, D, gpu)
    else:
        cache = tuple(torch.zeros(B, S, Hk * D, device=gpu, dtype=dtype) for _ in range(2))
    gone = torch.zeros(B, dtype=torch.int32, device=gpu)
    lens = torch.zeros(B, dtype=torch.int32, device=gpu)

    def held():  # what the caches hold, float64 [B, Hk, S, D]
        if q4:
            return Q.values(cache.k_codes, cache.k_scales, True, D)[0], Q.values(cache.v_codes, cache.v_scales, False, D)[0]
        return tuple(x.view(B, S, Hk, D).transpose(1, 2).double() for x in cache)

    rows = [[[] for _ in range(Hk)] for _ in range(B)]  # positions of the rows of each head
    seen = torch.zeros(B, dtype=torch.long)
    total = torch.zeros(B, Hk, S, device=gpu, dtype=torch.float64)
    t_total = torch.zeros_like(total)
    seed = 10

    def step(T, news):
        """``news``: how many of the T tokens are real; the first ones of a shorter prompt fall in front of the cache."""
        nonlocal seed, lens
        q, k, v = (rand((B, T, h * D), seed + i, dtype, gpu) for i, h in enumerate((H, Hk, Hk)))
        seed += 3
        lens = lens + torch.tensor(news, dtype=torch.int32, device=gpu)
        if q4:
            qr = fta.flash_qk_norm_rope_append_q4(q, k, v, cache, lens, H, cos, sin, qw, kw, num_kv_heads=Hk, position_offset=gone)
            o, lse = fta.flash_window_attn_decode_q4(qr, cache, lens, H, S, num_kv_heads=Hk)
            fta.flash_cache_weights(qr, cache, lse, lens, weights, H, S, num_kv_heads=Hk)
            ref = Q.attend(qr, cache, lens.tolist(), H, Hk, S, 0, D ** -0.5)
        else:
            qr = fta.flash_qk_norm_rope_append(q, k, v, *cache, lens, H, cos, sin, qw, kw, num_kv_heads=Hk, position_offset=gone)
            o, lse = fta.flash_window_attn_decode(qr, *cache, lens, H, S, num_kv_heads=Hk)
            fta.flash_cache_weights(qr, cache[0], lse, lens, weights, H, S, num_kv_heads=Hk)
            ref = R.cache(qr, *cache, lens.tolist(), H, Hk, S, 0, D ** -0.5)
        R.check({"o": o, "lse": lse}, ref, ("o", "lse"))
        pos = (lens + gone)[:, None] - T + torch.arange(T, device=gpu)
        exact = R.turned(q.double(), H, qw.double(), cos, sin, pos, 1e-6, False)
        assert ((qr.double() - exact).abs() <= R.half_step(dtype) * exact.abs() + 1e-4 * (1 + exact.abs())).all()
        ke = R.turned(k.double(), Hk, kw.double(), cos, sin, pos, 1e-6, False).unflatten(-1, (Hk, D))
        kk, _ = held()
        for b in range(B):
            for t in range(T - news[b], T):
                at = int(lens[b]) - T + t
                step_ = Q.values(cache.k_codes, cache.k_scales, True, D)[1][b, :, at] if q4 else 0.0
                off = (kk[b, :, at] - ke[b, t]).abs()
                assert (off <= step_ * 1.01 + 2 * R.half_step(dtype) * ke[b, t].abs() + 1e-4).all()
                for h in range(Hk):
                    rows[b][h].append(int(seen[b]))
                seen[b] += 1
        for b in range(B):
            n = int(lens[b])
            see = R.window_mask(T, n, n - T, S, 0, 0, gpu)
            for h in range(H):
                s = (qr[b].view(T, H, D)[:, h].double() @ kk[b, h // (H // Hk), :n].T * D ** -0.5).masked_fill(~see, -math.inf)
                x = torch.exp(s - lse[b, h, :, None].double().masked_fill(lse[b, h, :, None] == -math.inf, math.inf))
                total[b, h // (H // Hk), :n] += x.sum(0)
                t_total[b, h // (H // Hk), :n] += x.sum(0) * (Q.F4 + 1e-5)
        assert ((weights.double() - total).abs() <= t_total + 1e-30).all()

    step(100, prompts)
    step(1, [1, 1, 1])
    step(2, [2, 2, 2])
    for _ in range(2):  # evict, go on, evict again
        new, kept = fta.flash_cache_evict(cache, weights, lens, budget, 8, 2)
        for b in range(B):
            n = int(lens[b])
            for h in range(Hk):
                idx = [j for j in kept[b, h].tolist() if j >= 0]
                assert len(idx) == min(n, budget) == int(new[b]) and idx == sorted(set(idx))
                rows[b][h] = [rows[b][h][j] for j in idx]
                at = torch.tensor(idx, device=gpu)
                t, tt = total[b, h, at].clone(), t_total[b, h, at].clone()
                total[b, h] = 0
                t_total[b, h] = 0
                total[b, h, :len(idx)], t_total[b, h, :len(idx)] = t, tt
                if n > budget:
                    assert rows[b][h][:2] == [0, 1] and rows[b][h][-8:] == list(range(int(seen[b]) - 8, int(seen[b])))
        gone += lens - new
        lens = new
        for T in (1, 3, 1):
            step(T, [T] * B)


def test_offsets_of_each_request(gpu):
    """A device tensor of position offsets is the same as the numbers."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 3, 2, 4, 2, 64, 20
    q, k, v = (rand((B, T, h * D), i, BF, gpu) for i, h in enumerate((H, Hk, Hk)))
    cos, sin = _tables(200, D // 2, gpu)
    ln = torch.tensor([20, 2, 7], dtype=torch.int32, device=gpu)
    offs = [5, 170, -3]
    kc, vc = (torch.zeros(B, S, Hk * D, device=gpu, dtype=BF) for _ in range(2))
    got = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, ln, H, cos, sin, num_kv_heads=Hk,
                                        position_offset=torch.tensor(offs, dtype=torch.int32, device=gpu))
    for b in range(B):
        k1, v1 = (torch.zeros(1, S, Hk * D, device=gpu, dtype=BF) for _ in range(2))
        with pytest.warns(UserWarning) if offs[b] < 0 else _nothing():
            q1 = fta.flash_qk_norm_rope_append(q[b:b + 1], k[b:b + 1], v[b:b + 1], k1, v1, ln[b:b + 1], H, cos, sin,
                                               num_kv_heads=Hk, position_offset=offs[b])
        assert torch.equal(got[b], q1[0]) and torch.equal(kc[b], k1[0]) and torch.equal(vc[b], v1[0])


class _nothing:
    def __enter__(self):
        return None

    def __exit__(self, *a):
        return False


@pytest.mark.parametrize("q4", [False, True], ids=["16bit", "4bit"])
def test_captured_steps(gpu, q4):
    """A step (append, attention, weights) and an eviction as graphs, replayed while lengths and tokens
    change, with eager work in between; two graphs at once."""
    import flash_topk_attn_v2 as fta

    B, H, Hk, D, S = 2, 8, 2, 128, 700
    cos, sin = _tables(S + 100, D // 2, gpu)
    lens = torch.tensor([500, 300], dtype=torch.int32, device=gpu)
    q, k, v = (rand((B, 1, h * D), i, BF, gpu) for i, h in enumerate((H, Hk, Hk)))

    def fresh():
        if q4:
            return Q.cache(B, S, Hk, D, gpu, 3)
        return tuple(rand((B, S, Hk * D), 3 + i, BF, gpu) for i in (0, 1))

    def one(cache, weights, lens, q, k, v):
        if q4:
            qr = fta.flash_qk_norm_rope_append_q4(q, k, v, cache, lens, H, cos, sin, num_kv_heads=Hk)
            o, lse = fta.flash_window_attn_decode_q4(qr, cache, lens, H, 400, 4, num_kv_heads=Hk)
            fta.flash_cache_weights(qr, cache, lse, lens, weights, H, 400, 4, num_kv_heads=Hk)
        else:
            qr = fta.flash_qk_norm_rope_append(q, k, v, *cache, lens, H, cos, sin, num_kv_heads=Hk)
            o, lse = fta.flash_window_attn_decode(qr, *cache, lens, H, 400, 4, num_kv_heads=Hk)
            fta.flash_cache_weights(qr, cache[0], lse, lens, weights, H, 400, 4, num_kv_heads=Hk)
        return o, lse

    cache, weights = fresh(), torch.zeros(B, Hk, S, device=gpu)
    mine, w2 = fresh(), torch.zeros(B, Hk, S, device=gpu)  # the eager side's
    warm, w3 = fresh(), torch.zeros(B, Hk, S, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # first calls outside a capture, on what is not looked at
        one(warm, w3, lens, q, k, v)
        fta.flash_cache_evict(warm, w3, lens, 200, 10, 4)
    torch.cuda.current_stream().wait_stream(side)
    g, e = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = one(cache, weights, lens, q, k, v)
    with torch.cuda.graph(e):
        evicted = fta.flash_cache_evict(cache, weights, lens, 200, 10, 4)
    for i in range(6):
        for x, s in ((q, 0), (k, 1), (v, 2)):
            x.copy_(rand(x.shape, 100 + 3 * i + s, BF, gpu))
        if i == 4:  # the eviction, then on from there
            e.replay()
            new, kept = fta.flash_cache_evict(mine, w2, lens, 200, 10, 4)
            assert torch.equal(evicted[0], new) and torch.equal(evicted[1], kept)
            for x, y in zip(cache, mine):
                assert torch.equal(x, y)
            assert torch.equal(weights, w2)
            lens.copy_(new)
        lens += 1
        g.replay()
        want = one(mine, w2, lens, q, k, v)
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y), i
        assert torch.equal(weights, w2)


def test_another_stream(gpu):
    """The calls run on the current stream: work that it waits for is seen, and none of it on others."""
    import flash_topk_attn_v2 as fta

    B, H, Hk, D, S = 2, 8, 2, 64, 300
    c = Q.cache(B, S, Hk, D, gpu, 3)
    q = rand((B, 1, H * D), 1, BF, gpu)
    ln = torch.tensor([300, 150], dtype=torch.int32, device=gpu)
    want = fta.flash_window_attn_decode_q4(q, c, ln, H, S, num_kv_heads=Hk)
    s = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        x = torch.randn(2048, 2048, device=gpu)
        for _ in range(20):
            x = x @ x * 1e-3
        late.copy_(q)
        got = fta.flash_window_attn_decode_q4(late, c, ln, H, S, num_kv_heads=Hk)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_views(gpu):
    """q, k, v out of one projection; caches and weights that are parts of larger ones."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 2, 2, 4, 2, 96, 75
    qkv = rand((B, T, (H + 2 * Hk) * D), 1, FP, gpu)
    q, k, v = qkv.split([H * D, Hk * D, Hk * D], -1)
    big = Q.cache(B + 1, S, Hk + 1, D, gpu, 3)
    c = fta.Q4Cache(*(t[1:, 1:] for t in big))
    own = fta.Q4Cache(*(t.clone(memory_format=torch.contiguous_format) for t in c))
    first = [t[0].clone() for t in big]
    cos, sin = _tables(S, D // 2, gpu)
    ln = torch.tensor([75, 30], dtype=torch.int32, device=gpu)
    a = fta.flash_qk_norm_rope_append_q4(q, k, v, c, ln, H, cos, sin, num_kv_heads=Hk)
    b = fta.flash_qk_norm_rope_append_q4(q.contiguous(), k.contiguous(), v.contiguous(), own, ln, H, cos, sin, num_kv_heads=Hk)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(c, own))
    oa, ob = (fta.flash_window_attn_decode_q4(a, x, ln, H, S, num_kv_heads=Hk) for x in (c, own))
    assert torch.equal(oa[0], ob[0]) and torch.equal(oa[1], ob[1])
    wa, wb = torch.zeros(B, Hk + 2, S + 5, device=gpu)[:, 2:, 3:S + 3], torch.zeros(B, Hk, S, device=gpu)
    for x, w in ((c, wa), (own, wb)):
        fta.flash_cache_weights(a, x, oa[1], ln, w, H, S, num_kv_heads=Hk)
    assert torch.equal(wa, wb)
    ea, eb = (fta.flash_cache_evict(x, w, ln, 20, 3, 1) for x, w in ((c, wa), (own, wb)))
    assert torch.equal(ea[1], eb[1]) and torch.equal(wa, wb) and all(torch.equal(x, y) for x, y in zip(c, own))
    assert all(torch.equal(t[0], f) for t, f in zip(big, first))  # what is not in the view stays


@pytest.mark.parametrize("D", [64, 128])
def test_rows_past_32_bits(gpu, D):
    """Codes of one head of more than 4 GB: rows at both ends."""
    import flash_topk_attn_v2 as fta

    H, Hk, T = 4, 1, 2
    S = (1 << 32) // (D // 2) + 1000
    say("past 32 bits", D, S)
    c = fta.flash_q4_cache(1, S, Hk, D, gpu)
    small = Q.cache(1, 500, Hk, D, gpu, 3)
    for x, y in zip(c, small):
        x[:, :, -300:] = y[:, :, 200:]
        x[:, :, :200] = y[:, :, :200]
    q = rand((1, T, H * D), 1, BF, gpu)
    ln, ln2 = (torch.tensor([n], dtype=torch.int32, device=gpu) for n in (S, 500))
    o, lse = fta.flash_window_attn_decode_q4(q, c, ln, H, 298, 150, num_kv_heads=Hk)
    o2, lse2 = fta.flash_window_attn_decode_q4(q, small, ln2, H, 298, 150, num_kv_heads=Hk)
    ref = Q.attend(q, small, [500], H, Hk, 298, 150, D ** -0.5)
    for a, b in ((o, o2),):
        assert ((a.double() - b.double()).abs() <= 2 * ref["o_tol"]).all()
    assert ((lse.double() - lse2.double()).abs() <= 2 * ref["lse_tol"]).all()
    w, w2 = torch.zeros(1, Hk, S, device=gpu), torch.zeros(1, Hk, 500, device=gpu)
    fta.flash_cache_weights(q, c, lse, ln, w, H, 298, 150, num_kv_heads=Hk)
    fta.flash_cache_weights(q, small, lse2, ln2, w2, H, 298, 150, num_kv_heads=Hk)
    both = torch.cat((w[..., :200], w[..., -300:]), -1)
    assert ((both - w2).abs() <= 4 * Q.F4 * w2 + 1e-30).all() and int((w != 0).sum()) == int((w2 != 0).sum())


def test_the_same_bits_every_run(gpu):
    import flash_topk_attn_v2 as fta

    B, H, Hk, D, S = 3, 8, 2, 128, 3000
    c = Q.cache(B, S, Hk, D, gpu, 3)
    q = rand((B, 100, H * D), 1, BF, gpu)
    ln = torch.tensor([S, 2000, 99], dtype=torch.int32, device=gpu)
    first = None
    for _ in range(3):
        o, lse = fta.flash_window_attn_decode_q4(q, c, ln, H, S, num_kv_heads=Hk)
        w = torch.zeros(B, Hk, S, device=gpu)
        fta.flash_cache_weights(q, c, lse, ln, w, H, S, num_kv_heads=Hk)
        new, kept = fta.flash_cache_evict(fta.Q4Cache(*(t.clone() for t in c)), w.clone(), ln, 500, 20, 4)
        now = (o, lse, w, new, kept)
        first = first or now
        assert all(torch.equal(x, y) for x, y in zip(first, now))


def test_refusals(gpu):
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 2, 1, 4, 2, 64, 32
    q, k, v = (rand((B, T, h * D), i, BF, gpu) for i, h in enumerate((H, Hk, Hk)))
    cos, sin = _tables(S, D // 2, gpu)
    ln = torch.tensor([32, 5], dtype=torch.int32, device=gpu)
    c = Q.cache(B, S, Hk, D, gpu, 3)
    w = torch.zeros(B, Hk, S, device=gpu)
    kc, vc = (rand((B, S, Hk * D), 5 + i, BF, gpu) for i in (0, 1))
    lse = torch.zeros(B, H, T, device=gpu)
    one = fta.Q4Cache(*(t[:1].expand(B, -1, -1, -1) for t in c))
    same = fta.Q4Cache(c.k_codes, c.k_scales, c.k_codes, c.v_scales)
    wide = Q.cache(B, S, Hk, 128, gpu, 3)
    byrow = fta.Q4Cache(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in c))
    off = torch.zeros(B * Hk * S * 32 + 16, dtype=torch.uint8, device=gpu)[8:-8].view(B, Hk, S, 32)

    def append(**x):
        a = dict(q=q, k=k, v=v, cache=c, cache_lens=ln, num_heads=H, cos=cos, sin=sin, num_kv_heads=Hk)
        return lambda: fta.flash_qk_norm_rope_append_q4(**{**a, **x})

    def decode(**x):
        a = dict(q=q, cache=c, cache_lens=ln, num_heads=H, window_left=5, num_kv_heads=Hk)
        return lambda: fta.flash_window_attn_decode_q4(**{**a, **x})

    def weigh(**x):
        a = dict(q=q, cache=c, lse=lse, cache_lens=ln, weights=w, num_heads=H, window_left=5, num_kv_heads=Hk)
        return lambda: fta.flash_cache_weights(**{**a, **x})

    def evict(**x):
        a = dict(cache=c, weights=w, cache_lens=ln, budget=8)
        return lambda: fta.flash_cache_evict(**{**a, **x})

    grad = q.clone().requires_grad_(True)
    bad = [
        append(cache=tuple(c)), append(cache=wide), append(cache=one), append(cache=same), append(cache=byrow),
        append(cache=c._replace(k_codes=off)), append(cache=c._replace(k_scales=c.k_scales.float())),
        append(cache_lens=ln.long()), append(cache_lens=ln[:1]), append(v=v.half()), append(q=grad), append(q=q.float()),
        append(position_offset=0.5), append(position_offset=ln.long()), append(position_offset=ln[:1]),
        append(position_offset=ln.cpu()), append(q=q.cpu()), append(cache=fta.Q4Cache(*(t.cpu() for t in c))),
        append(num_heads=3), append(eps=0.0),
        decode(cache=wide), decode(cache=(kc, vc)), decode(window_left=-1), decode(num_sinks=-1), decode(window_left=1.5),
        decode(scale=0.0), decode(scale=math.inf), decode(q=grad), decode(q=q[:, :0]), decode(cache=byrow), decode(q=q[0]),
        decode(cache_lens=ln.cpu()), decode(num_kv_heads=3),
        weigh(lse=lse[..., :0]), weigh(lse=lse.half()), weigh(weights=w.double()), weigh(weights=w[..., :-1]),
        weigh(weights=w[:, :1].expand(-1, Hk, -1)), weigh(weights=w[0]), weigh(cache=kc.half()), weigh(cache=kc[:, :, :-16]),
        weigh(cache=(kc, vc)), weigh(q=grad), weigh(weights=w.cpu()), weigh(window_left=-1),
        weigh(weights=w.transpose(1, 2).contiguous().transpose(1, 2)),
        evict(budget=0), evict(budget=S + 1), evict(budget=8, num_recent=5, num_sinks=4), evict(num_recent=-1),
        evict(budget=2.5), evict(weights=w[..., :-1]), evict(weights=w.half()), evict(cache=one), evict(cache=same),
        evict(cache=kc), evict(cache=(kc, kc)), evict(cache=(kc, vc[:, :-1])), evict(cache=(kc, vc.half())),
        evict(cache=(kc[:1].expand(B, -1, -1), vc)), evict(cache_lens=ln.long()), evict(out=c), evict(out=(c, w)),
        evict(out=((kc, vc), w.clone())), evict(out=(wide, w.clone())), evict(out=(Q.cache(B, 4, Hk, D, gpu, 1), w[..., :4].clone())),
        evict(cache=(kc, vc), out=((kc.clone(), vc), w.clone())), evict(cache=(kc, vc), out=((kc.half(), vc.half()), w.clone())),
        lambda: fta.flash_q4_cache_read(c, 65, BF), lambda: fta.flash_q4_cache_read(c, 128, BF),
        lambda: fta.flash_q4_cache_read(c, D, torch.float32), lambda: fta.flash_q4_cache_read((kc, vc), D, BF),
        lambda: fta.flash_q4_cache(0, 1, 1, 64, gpu), lambda: fta.flash_q4_cache(1, 1, 1, 65, gpu),
        lambda: fta.flash_q4_cache(1, 1, 1, 512, gpu),
    ]
    before = [t.clone() for t in (*c, w, kc, vc)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            say("not refused:", i)
    assert all(torch.equal(x, y) for x, y in zip(before, (*c, w, kc, vc)))
    with torch.no_grad():  # and what is not refused
        append(q=grad)()
        decode(q=grad)()
        weigh(q=grad)()
    evict()()
