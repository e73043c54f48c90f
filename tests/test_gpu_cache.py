"""Attention of new tokens over K/V caches, with a window and sinks or behind a shared
prefix, against its definition in float64, and the operators together as they are used."""

import math

import pytest
import torch

import _operators_ref as R
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _state(dev, dtype, B, T, H, Hk, D, S, lens, seed=3):
    q = rand((B, T, H * D), seed, dtype, dev)
    kc, vc = (rand((B, S, Hk * D), seed + i, dtype, dev) for i in (1, 2))
    if lens is None:
        lens = torch.randint(T, S + 1, (B,), generator=torch.Generator().manual_seed(seed)).tolist()
    return q, kc, vc, torch.tensor(lens, dtype=torch.int32, device=dev)


# dtype, B, T, H, Hk, D, S, left, sinks, lens
WINDOW = [
    (BF, 1, 1, 1, 1, 64, 1, 0, 0, [1]),
    (BF, 4, 1, 8, 2, 128, 100, 20, 4, [100, 1, 0, 57]),
    (FP, 3, 2, 4, 4, 64, 333, 100, 0, None),
    (BF, 2, 1, 8, 1, 256, 700, 10000, 3, None),
    (FP, 2, 5, 16, 2, 80, 300, 31, 33, [3, 300]),       # fewer tokens than new ones: rows that see nothing
    (BF, 1, 1, 32, 8, 128, 3000, 2047, 4, [3000]),      # many parts
    (BF, 1, 1, 2, 2, 64, 9000, 8191, 100, [8999]),
    (FP, 70, 1, 8, 8, 128, 257, 128, 1, None),
    (BF, 2, 40, 4, 2, 64, 128, 17, 5, [128, 60]),       # several row tiles
    (FP, 3, 3, 33, 1, 96, 90, 90, 0, None),             # 99 rows on one K/V head
    (BF, 2, 1, 4, 2, 16, 50, 0, 0, [-4, 1000]),         # lengths outside the cache are clamped
    (BF, 2, 3, 4, 2, 128, 200, 5, 200, [200, 66]),      # every key a sink
]


@pytest.mark.parametrize("case", WINDOW, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_window_decode(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, B, T, H, Hk, D, S, left, sinks, lens = case
    say("wdecode", case)
    q, kc, vc, ln = _state(gpu, dtype, B, T, H, Hk, D, S, lens)
    o, lse = fta.flash_window_attn_decode(q, kc, vc, ln, H, left, sinks, num_kv_heads=Hk)
    ref = R.cache(q, kc, vc, ln.tolist(), H, Hk, left, sinks, D ** -0.5)
    R.check({"o": o, "lse": lse}, ref, ("o", "lse"), str(case))


# dtype, B, T, H, Hk, D, P, S, lens
PREFIX = [
    (BF, 1, 1, 1, 1, 64, 1, 1, [1]),
    (FP, 3, 2, 4, 2, 64, 100, 40, None),
    (BF, 8, 1, 32, 8, 128, 1000, 64, None),
    (FP, 40, 1, 8, 2, 80, 333, 17, None),
    (BF, 33, 3, 16, 2, 128, 2048, 100, None),            # 792 rows on each K/V head
    (FP, 2, 1, 4, 2, 256, 500, 300, None),
    (BF, 4, 2, 4, 4, 128, 64, 30, [0, 1, 30, 2]),        # idle requests see the prefix alone
    (BF, 2, 1, 4, 2, 64, 0, 30, [0, 30]),                # no prefix
    (FP, 1, 1, 8, 1, 96, 9000, 5, [5]),
]


@pytest.mark.parametrize("case", PREFIX, ids=lambda c: "-".join(str(x) for x in c[1:8]))
def test_prefix_decode(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, B, T, H, Hk, D, P, S, lens = case
    say("prefix", case)
    q, kc, vc, ln = _state(gpu, dtype, B, T, H, Hk, D, S, lens)
    kp, vp = (rand((P, Hk * D), 20 + i, dtype, gpu) for i in (0, 1))
    o, lse = fta.flash_prefix_attn_decode(q, kp, vp, kc, vc, ln, H, num_kv_heads=Hk)
    ref = R.cache(q, kc, vc, ln.tolist(), H, Hk, S, 0, D ** -0.5, kp, vp)
    R.check({"o": o, "lse": lse}, ref, ("o", "lse"), str(case))


def test_prefix_is_the_same_as_a_copy_in_every_cache(gpu):
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, P, S = 5, 2, 8, 2, 128, 200, 60
    q, kc, vc, ln = _state(gpu, BF, B, T, H, Hk, D, S, None)
    kp, vp = (rand((P, Hk * D), 20 + i, BF, gpu) for i in (0, 1))
    o, lse = fta.flash_prefix_attn_decode(q, kp, vp, kc, vc, ln, H, num_kv_heads=Hk)
    whole = [torch.cat((p.expand(B, -1, -1), c), 1) for p, c in ((kp, kc), (vp, vc))]
    o2, lse2 = fta.flash_window_attn_decode(q, *whole, ln + P, H, P + S, num_kv_heads=Hk)
    ref = R.cache(q, kc, vc, ln.tolist(), H, Hk, S, 0, D ** -0.5, kp, vp)
    assert ((o.double() - o2.double()).abs() <= 2 * ref["o_tol"]).all()
    assert ((lse.double() - lse2.double()).abs() <= 2 * ref["lse_tol"]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_unseen_rows_may_hold_anything(gpu, D):
    """Rows past the lengths, and between the sinks and the window, hold NaN and infinities."""
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, S, left, sinks, lens = 3, 2, 4, 2, 400, 50, 5, [400, 0, 207]
    q, kc, vc, ln = _state(gpu, BF, B, T, H, Hk, D, S, lens)
    clean = fta.flash_window_attn_decode(q, kc, vc, ln, H, left, sinks, num_kv_heads=Hk)
    for b in range(B):
        for x, bad in ((kc, math.nan), (vc, math.inf)):
            x[b, lens[b]:] = bad
            x[b, sinks:max(sinks, lens[b] - T - left)] = bad
    dirty = fta.flash_window_attn_decode(q, kc, vc, ln, H, left, sinks, num_kv_heads=Hk)
    for x, y in zip(clean, dirty):
        assert torch.equal(x, y)
    assert (dirty[0][1] == 0).all() and (dirty[1][1] == -math.inf).all()
    kp, vp = (rand((70, Hk * D), 30 + i, BF, gpu) for i in (0, 1))
    k2, v2 = (torch.where(x.isfinite(), x, torch.zeros_like(x)) for x in (kc, vc))
    k3, v3 = k2.clone(), v2.clone()
    for b in range(B):
        k3[b, lens[b]:], v3[b, lens[b]:] = math.inf, math.nan
    for x, y in zip(fta.flash_prefix_attn_decode(q, kp, vp, k2, v2, ln, H, num_kv_heads=Hk),
                    fta.flash_prefix_attn_decode(q, kp, vp, k3, v3, ln, H, num_kv_heads=Hk)):
        assert torch.equal(x, y)


def test_long_cache_offsets(gpu):
    """Batch and token offsets past 2^32 bytes and 2^31 elements."""
    import flash_topk_attn_v2 as fta

    B, S, H, D = 2, (1 << 24) + 100, 1, 64
    q = rand((B, 1, H * D), 1, BF, gpu)
    kc = torch.empty(B, S, H * D, device=gpu, dtype=BF)
    vc = torch.empty(B, S, H * D, device=gpu, dtype=BF)
    lens, left = [S, S - 37], 300
    for b, n in enumerate(lens):  # only what is seen
        kc[b, n - left - 1:n] = rand((left + 1, H * D), 2 + b, BF, gpu)
        vc[b, n - left - 1:n] = rand((left + 1, H * D), 4 + b, BF, gpu)
        kc[b, :3], vc[b, :3] = rand((3, H * D), 6 + b, BF, gpu), rand((3, H * D), 8 + b, BF, gpu)
    o, lse = fta.flash_window_attn_decode(q, kc, vc, torch.tensor(lens, dtype=torch.int32, device=gpu), H, left, 3)
    for b, n in enumerate(lens):
        at = torch.cat((torch.arange(3), torch.arange(n - left - 1, n))).to(gpu)
        r = R.attend(q[b].double(), kc[b, at].double(), vc[b, at].double(),
                     torch.ones(1, at.numel(), device=gpu, dtype=torch.bool), D ** -0.5, BF)
        assert ((o[b].double() - r["o"]).abs() <= r["o_tol"]).all()
        assert ((lse[b, 0].double() - r["lse"]).abs() <= r["lse_tol"]).all()


def test_layouts_and_streams(gpu):
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 3, 2, 4, 2, 64, 150
    q, kc, vc, ln = _state(gpu, FP, B, T, H, Hk, D, S, None)
    both = torch.empty(S, B, 2 * Hk * D, device=gpu, dtype=FP)
    kv, vv = both.transpose(0, 1).split(Hk * D, -1)
    kv.copy_(kc)
    vv.copy_(vc)
    kp, vp = (rand((90, Hk * D), 30 + i, FP, gpu) for i in (0, 1))
    pp = torch.cat((kp, vp), -1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = [*fta.flash_window_attn_decode(q, kc, vc, ln, H, 40, 3, num_kv_heads=Hk),
            *fta.flash_prefix_attn_decode(q, kp, vp, kc, vc, ln, H, num_kv_heads=Hk)]
    with torch.cuda.stream(side):
        got = [*fta.flash_window_attn_decode(q, kv, vv, ln, H, 40, 3, num_kv_heads=Hk),
               *fta.flash_prefix_attn_decode(q, *pp.split(Hk * D, -1), kv, vv, ln, H, num_kv_heads=Hk)]
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    shared = kc[:1].expand(B, -1, -1)  # one cache for all: read only, so it may be expanded
    a = fta.flash_window_attn_decode(q, shared, shared, ln, H, 40, 3, num_kv_heads=Hk)
    b = fta.flash_window_attn_decode(q, shared.contiguous(), shared.contiguous(), ln, H, 40, 3, num_kv_heads=Hk)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def _tables(P, Rc, dev):
    inv = 10000.0 ** (-torch.arange(0, Rc, 2, dtype=torch.float64) / Rc)
    a = torch.arange(P, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(dev), a.sin().float().to(dev)


def _layer(B, N, H, Hk, D, dev, seed):
    x = [rand((B, N, n * D), seed + i, BF, dev) for i, n in enumerate((H, Hk, Hk))]
    w = [1 + 0.1 * rand((D,), seed + 5 + i, torch.float32, dev) for i in range(2)]
    return x, w


def test_a_layer_trained_and_then_served(gpu):
    """Preparation -> window attention over whole sequences, with gradients down to the norm
    weights, and the same sequences served token by token through the caches: the served
    rows are the trained ones within the bounds of both."""
    import flash_topk_attn_v2 as fta

    B, N, H, Hk, D, left, sinks, start = 2, 150, 4, 2, 64, 30, 4, 100
    (q, k, v), (qw, kw) = _layer(B, N, H, Hk, D, gpu, 60)
    cos, sin = _tables(N, D, gpu)
    leaves = [x.requires_grad_(True) for x in (q, k, v, qw, kw)]
    qp, kp = fta.flash_qk_norm_rope(q, k, H, cos, sin, qw, kw, num_kv_heads=Hk)
    o, lse = fta.flash_window_attn(qp, kp, v, H, (left, 0), sinks, num_kv_heads=Hk)
    do = rand((B, N, H * D), 70, BF, gpu)
    grads = torch.autograd.grad(o, leaves, do)
    ref = R.window(qp.detach(), kp.detach(), v.detach(), H, Hk, left, 0, sinks, D ** -0.5, None, do)
    R.check({"o": o, "lse": lse, "dv": grads[2]}, ref, ("o", "lse", "dv"))
    with torch.no_grad():
        # the chain: the preparation's backward on the attention's gradients
        dqp, dkp = torch.zeros_like(qp), torch.zeros_like(kp)
    qp2, kp2 = (x.detach().requires_grad_(True) for x in (qp, kp))
    o2, _ = fta.flash_window_attn(qp2, kp2, v.detach(), H, (left, 0), sinks, num_kv_heads=Hk)
    dqp, dkp = torch.autograd.grad(o2, (qp2, kp2), do)
    a, b = fta.flash_qk_norm_rope(q, k, H, cos, sin, qw, kw, num_kv_heads=Hk)
    for x, y in zip(torch.autograd.grad((a, b), (q, k, qw, kw), (dqp, dkp)), (grads[0], grads[1], grads[3], grads[4])):
        assert torch.equal(x, y)
    with torch.no_grad():
        kc, vc = (torch.full((B, N, Hk * D), math.nan, device=gpu, dtype=BF) for _ in range(2))
        lens = torch.full((B,), start, dtype=torch.int32, device=gpu)
        fta.flash_qk_norm_rope_append(q[:, :start], k[:, :start], v[:, :start], kc, vc, lens, H, cos, sin, qw, kw,
                                      num_kv_heads=Hk)
        assert torch.equal(kc[:, :start], kp.detach()[:, :start])
        at = start
        while at < N:
            T = min(3, N - at)
            lens += T
            qn = fta.flash_qk_norm_rope_append(q[:, at:at + T], k[:, at:at + T], v[:, at:at + T], kc, vc, lens, H, cos,
                                               sin, qw, kw, num_kv_heads=Hk)
            assert torch.equal(qn, qp.detach()[:, at:at + T])
            on, ln = fta.flash_window_attn_decode(qn, kc, vc, lens, H, left, sinks, num_kv_heads=Hk)
            assert ((on.double() - ref["o"][:, at:at + T]).abs() <= ref["o_tol"][:, at:at + T]).all()
            assert ((ln.double() - ref["lse"][:, :, at:at + T]).abs() <= ref["lse_tol"][:, :, at:at + T]).all()
            at += T


def test_prepared_queries_into_the_sparse_attention(gpu):
    """The preparation in front of the framework's own pipeline, and its gradients through it."""
    import flash_topk_attn_v2 as fta

    B, N, H, D = 1, 512, 2, 64
    (q, k, v), (qw, kw) = _layer(B, N, H, H, D, gpu, 90)
    cos, sin = _tables(N, D, gpu)
    leaves = [x.requires_grad_(True) for x in (q, k, qw, kw)]
    qp, kp = fta.flash_qk_norm_rope(q, k, H, cos, sin, qw, kw)
    idx, _, avg = fta.flash_topk_score(qp.detach(), kp.detach(), H, 64, 8)  # all eight blocks: full attention
    merged, counts, _ = fta.build_qblock_topk_indices(idx, 32, (0, 0), avg)
    o, lse = fta.flash_topk_attn(qp, kp, v, merged, counts, H, 32, 64)
    ow, lw = fta.flash_window_attn(qp, kp, v, H, (N, N))
    ref = R.window(qp.detach(), kp.detach(), v, H, H, N, N, 0, D ** -0.5)
    R.check({"o": o, "lse": lse}, ref, ("o", "lse"), "sparse")
    R.check({"o": ow, "lse": lw}, ref, ("o", "lse"), "window")
    do = rand((B, N, H * D), 99, BF, gpu)
    for g in torch.autograd.grad(o, leaves, do):
        assert g.isfinite().all() and (g != 0).any()


def test_serving_step_in_a_graph(gpu):
    """One captured step -- lengths up by one, append, both attentions -- replayed while the
    requests grow, another graph of the same shapes captured beside it, eager work between."""
    import flash_topk_attn_v2 as fta

    B, H, Hk, D, S, P = 3, 8, 2, 128, 300, 130
    (q0, k0, v0), (qw, kw) = _layer(B, 40, H, Hk, D, gpu, 120)
    cos, sin = _tables(P + S, D, gpu)
    kp, vp = (rand((P, Hk * D), 140 + i, BF, gpu) for i in (0, 1))
    q, k, v = (torch.zeros(B, 1, n * D, device=gpu, dtype=BF) for n in (H, Hk, Hk))
    base_k, base_v = (rand((B, S, Hk * D), 150 + i, BF, gpu) for i in (0, 1))
    start = torch.tensor([250, 3, 77], dtype=torch.int32, device=gpu)

    def step(kc, vc, lens):
        lens += 1
        qn = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos, sin, qw, kw, num_kv_heads=Hk, position_offset=P)
        return (*fta.flash_window_attn_decode(qn, kc, vc, lens, H, 100, 4, num_kv_heads=Hk),
                *fta.flash_prefix_attn_decode(qn, kp, vp, kc, vc, lens, H, num_kv_heads=Hk))

    with torch.no_grad():
        sets = []
        for _ in range(2):
            state = (base_k.clone(), base_v.clone(), start.clone())
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(*state)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*state)
            for x, y in zip(state, (base_k, base_v, start)):
                x.copy_(y)
            sets.append((graph, out, state))
        eager = (base_k.clone(), base_v.clone(), start.clone())
        for i in range(4):
            for x, y in zip((q, k, v), (q0, k0, v0)):
                x.copy_(y[:, i:i + 1])
            for graph, _, _ in sets:
                graph.replay()
            torch.cuda.synchronize()
            want = step(*eager)
            for _, out, state in sets:
                for x, y in zip((*want, *eager), (*out, *state)):
                    assert torch.equal(x, y), i


def test_refusals(gpu):
    import flash_topk_attn_v2 as fta

    B, T, H, Hk, D, S = 2, 2, 4, 2, 64, 20
    q, kc, vc, ln = _state(gpu, BF, B, T, H, Hk, D, S, None)
    good = dict(q=q, k_cache=kc, v_cache=vc, cache_lens=ln, num_heads=H, num_kv_heads=Hk)
    bad = [dict(q=q[0]), dict(q=q.float()), dict(q=q[:1]), dict(q=q[:, :0]), dict(k_cache=kc.half()), dict(v_cache=vc[:, :3]),
           dict(num_heads=3), dict(num_kv_heads=4), dict(num_kv_heads=3), dict(cache_lens=ln.long()), dict(cache_lens=ln.cpu()),
           dict(scale=0.0), dict(scale=float("nan")), dict(k_cache=kc.transpose(1, 2)),
           dict(k_cache=torch.zeros(B, S, 2 * Hk * D, device=gpu, dtype=BF)[..., ::2])]
    win, pre = dict(window_left=5, num_sinks=2), dict(k_prefix=kc[0], v_prefix=vc[0])
    fta.flash_window_attn_decode(**good, **win)
    fta.flash_prefix_attn_decode(**good, **pre)
    for b in bad:
        with pytest.raises(ValueError):
            fta.flash_window_attn_decode(**(good | b), **win)
        with pytest.raises(ValueError):
            fta.flash_prefix_attn_decode(**(good | b), **pre)
    for b in (dict(window_left=-1), dict(num_sinks=-1)):
        with pytest.raises(ValueError):
            fta.flash_window_attn_decode(**good, **(win | b))
    for b in (dict(k_prefix=kc), dict(v_prefix=vc[0, :3]), dict(k_prefix=kc[0].half()), dict(k_prefix=kc[0].cpu()),
              dict(k_prefix=kc[0, :, :64]), dict(k_prefix=None)):
        with pytest.raises(ValueError):
            fta.flash_prefix_attn_decode(**good, **(pre | b))
    g = good | dict(q=q.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="not differentiable"):
        fta.flash_window_attn_decode(**g, **win)
    with torch.no_grad():
        fta.flash_window_attn_decode(**g, **win)


@pytest.mark.parametrize("case", range(12))
def test_drawn_shapes(gpu, case):
    """Shapes over the whole range, odd ones among them, both forms on the same caches."""
    import random

    import flash_topk_attn_v2 as fta

    r = random.Random(100 + case)
    dtype, D = r.choice([BF, FP]), r.choice([16, 64, 80, 128, 176, 256])
    Hk, G = r.choice([1, 2, 3, 8]), r.choice([1, 2, 3, 4, 8])
    B, T, S, P = r.choice([1, 2, 3, 20]), r.choice([1, 1, 2, 5, 9]), r.randrange(1, 900), r.randrange(1, 900)
    left, sinks = r.randrange(0, 400), r.choice([0, 1, 4, 33, 150])
    lens = [r.randrange(0, S + 1) for _ in range(B)]
    say("cache drawn", case, dtype, B, T, Hk * G, Hk, D, S, P, left, sinks, lens)
    q, kc, vc, ln = _state(gpu, dtype, B, T, Hk * G, Hk, D, S, lens, seed=2000 + case)
    kp, vp = (rand((P, Hk * D), 3000 + i, dtype, gpu) for i in (0, 1))
    o, lse = fta.flash_window_attn_decode(q, kc, vc, ln, Hk * G, left, sinks, num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, R.cache(q, kc, vc, lens, Hk * G, Hk, left, sinks, D ** -0.5), ("o", "lse"))
    o, lse = fta.flash_prefix_attn_decode(q, kp, vp, kc, vc, ln, Hk * G, num_kv_heads=Hk)
    R.check({"o": o, "lse": lse}, R.cache(q, kc, vc, lens, Hk * G, Hk, S, 0, D ** -0.5, kp, vp), ("o", "lse"))
