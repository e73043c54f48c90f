"""Sliding-window attention with sinks against its definition in float64: forward and
backward, masks that leave little, ragged and empty sequences, layouts, graphs."""

import math

import pytest
import torch

import _operators_ref as R
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16

# dtype, B, N, H, Hk, D, left, right, sinks, lens
CASES = [
    (BF, 1, 1, 1, 1, 64, 0, 0, 0, None),
    (BF, 2, 1, 4, 2, 128, 5, 5, 3, [1, 0]),
    (FP, 1, 17, 2, 1, 16, 3, 0, 1, None),
    (BF, 1, 64, 2, 2, 64, 0, 0, 0, None),        # only itself
    (FP, 2, 65, 3, 1, 32, 0, 0, 1, None),
    (BF, 1, 300, 4, 2, 128, 5, 0, 3, None),
    (FP, 1, 300, 4, 4, 128, 31, 2, 40, None),    # sinks that reach into the band
    (BF, 2, 333, 8, 2, 80, 64, 64, 16, [333, 70]),
    (FP, 2, 513, 6, 2, 64, 100, 0, 130, [200, 513]),  # three heads a group, sinks over three tiles
    (BF, 1, 700, 2, 1, 96, 10000, 0, 4, None),   # plain causal
    (FP, 1, 450, 2, 2, 48, 10000, 10000, 0, None),  # everything
    (BF, 1, 450, 4, 1, 144, 0, 200, 0, None),    # looks ahead only
    (BF, 3, 200, 4, 2, 256, 50, 0, 4, [0, 1, 200]),
    (FP, 1, 390, 2, 1, 256, 127, 31, 70, None),
    (BF, 1, 200, 2, 2, 112, 20, 0, 1000, None),  # every key is a sink
    (FP, 2, 129, 16, 1, 64, 63, 0, 0, None),     # sixteen heads on one
    (BF, 1, 2100, 2, 1, 64, 40, 0, 5, None),     # the sinks' walk in many parts
    (BF, 2, 500, 4, 4, 64, 64, 0, 4, [-3, 1000]),  # lengths outside the sequence are clamped
]


def _inputs(dev, dtype, B, N, H, Hk, D, seed=7):
    q, do = (rand((B, N, H * D), seed + i, dtype, dev) for i in (0, 1))
    k, v = (rand((B, N, Hk * D), seed + i, dtype, dev) for i in (2, 3))
    return q, k, v, do


def _run(q, k, v, do, H, Hk, win, sinks, lens=None, scale=None):
    import flash_topk_attn_v2 as fta

    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    o, lse = fta.flash_window_attn(q, k, v, H, win, sinks, scale=scale, num_kv_heads=Hk, seq_lens=lens)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {"o": o.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


ALL = ("o", "lse", "dq", "dk", "dv")


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[1:9]))
def test_forward_and_gradients(gpu, case):
    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    say("window", case)
    q, k, v, do = _inputs(gpu, dtype, B, N, H, Hk, D)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)
    got = _run(q, k, v, do, H, Hk, (left, right), sinks, ln)
    ref = R.window(q, k, v, H, Hk, left, right, sinks, D ** -0.5, lens, do)
    R.check(got, ref, ALL, str(case))


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,left,sinks", [
    (BF, 1, 4200, 32, 8, 128, 500, 4), (FP, 2, 4100, 16, 16, 64, 127, 1), (BF, 1, 4099, 32, 4, 64, 1023, 70),
    (FP, 4, 1000, 16, 16, 16, 40, 900), (BF, 5, 600, 32, 16, 256, 9, 500)])  # more tiles of sinks than parts for each
def test_grids_that_fill_the_card(gpu, dtype, B, N, H, Hk, D, left, sinks):
    """Many workgroups, whose heads share K and V."""
    say("window large", dtype, B, N, H, Hk, D)
    q, k, v, do = _inputs(gpu, dtype, B, N, H, Hk, D)
    got = _run(q, k, v, do, H, Hk, (left, 0), sinks)
    R.check(got, R.window(q, k, v, H, Hk, left, 0, sinks, D ** -0.5, None, do), ALL)


def test_large_scores_and_scale(gpu):
    """Scores of hundreds: the running maximum moves by far more than a rounding-free step.

    With inputs four times and a scale three times the usual, scores are 48 times larger,
    and so is the exponent's error: F grows to 48 F.
    """
    q, k, v, do = _inputs(gpu, BF, 1, 500, 2, 2, 64)
    q, k = q * 4, k * 4
    got = _run(q, k, v, do, 2, 2, (100, 0), 4, scale=3 / 8)
    old, R.F = R.F, 48 * R.F
    try:
        ref = R.window(q, k, v, 2, 2, 100, 0, 4, 3 / 8, None, do)
    finally:
        R.F = old
    R.check(got, ref, ALL)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_padding_may_hold_anything(gpu, D):
    """NaN and infinities at and past seq_lens change nothing, and their gradients are zero."""
    B, N, H, Hk, lens = 3, 300, 4, 2, [130, 0, 299]
    q, k, v, do = _inputs(gpu, BF, B, N, H, Hk, D)
    ln = torch.tensor(lens, dtype=torch.int32, device=gpu)
    clean = _run(q, k, v, do, H, Hk, (70, 3), 5, ln)
    for x, bad in zip((q, k, v, do), (math.nan, math.inf, -math.inf, math.nan)):
        for b in range(B):
            x[b, lens[b]:] = bad
    dirty = _run(q, k, v, do, H, Hk, (70, 3), 5, ln)
    for n in ALL:
        assert torch.equal(clean[n], dirty[n]), n
    for b in range(B):
        for n in ("o", "dq", "dk", "dv"):
            assert (dirty[n][b, lens[b]:] == 0).all()
        assert (dirty["lse"][b, :, lens[b]:] == -math.inf).all()


def test_layouts(gpu):
    """Views of a packed tensor, an expanded batch, unaligned rows: the results of dense copies."""
    import flash_topk_attn_v2 as fta

    B, N, H, Hk, D = 2, 210, 4, 2, 64
    packed = rand((B, N, (H + 2 * Hk) * D), 3, BF, gpu)
    q, k, v = packed.split((H * D, Hk * D, Hk * D), -1)
    do = rand((B, N, H * D), 5, BF, gpu)
    want = _run(q.contiguous(), k.contiguous(), v.contiguous(), do, H, Hk, (40, 0), 4)
    got = _run(q, k, v, do, H, Hk, (40, 0), 4)
    shifted = torch.empty(B, N, H * D + 3, device=gpu, dtype=BF)[..., 3:]  # rows off the 16-byte grid
    shifted.copy_(q)
    got2 = _run(shifted, k, v, do, H, Hk, (40, 0), 4)
    rows = torch.zeros(N, B, H * D, device=gpu, dtype=BF).transpose(0, 1)  # token-major gradient
    rows.copy_(do)
    got3 = _run(q, k, v, rows, H, Hk, (40, 0), 4)
    for n in ALL:
        assert torch.equal(want[n], got[n]) and torch.equal(want[n], got2[n]) and torch.equal(want[n], got3[n]), n
    # one K/V for the whole batch: its gradient is the batch's sum
    k1, v1 = (x[:1].contiguous().requires_grad_(True) for x in (k, v))
    o, _ = fta.flash_window_attn(q, k1.expand(B, -1, -1), v1.expand(B, -1, -1), H, (40, 0), 4, num_kv_heads=Hk)
    dk, dv = torch.autograd.grad(o, (k1, v1), do)
    dense = _run(q.contiguous(), k[:1].repeat(B, 1, 1), v[:1].repeat(B, 1, 1), do, H, Hk, (40, 0), 4)
    assert torch.equal(o.detach(), dense["o"])
    for got, n in ((dk, "dk"), (dv, "dv")):
        x = dense[n].float()
        assert ((got.float() - x.sum(0, keepdim=True)).abs() <= R.half_step(BF) * x.abs().sum(0)).all()


def test_wide_token_strides(gpu):
    """A token stride past 2^24 elements, which the 32-bit lane offsets do not span."""
    N, H, D, stride = 70, 1, 64, (1 << 24) + 8
    base = torch.zeros(N * stride + D, device=gpu, dtype=BF)
    wide = base.as_strided((1, N, H * D), (N * stride, stride, 1))
    q, k, v, do = _inputs(gpu, BF, 1, N, H, H, D)
    want = _run(q, k, v, do, H, H, (20, 0), 2)
    wide.copy_(k)
    got = _run(q, wide, v, do, H, H, (20, 0), 2)
    for n in ALL:
        assert torch.equal(want[n], got[n]), n
    wide.copy_(q)
    got = _run(wide, k, v, do, H, H, (20, 0), 2)
    for n in ALL:
        assert torch.equal(want[n], got[n]), n


def test_same_bits_and_other_stream(gpu):
    q, k, v, do = _inputs(gpu, FP, 2, 700, 4, 2, 64)
    want = _run(q, k, v, do, 4, 2, (90, 0), 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, 4, 2, (90, 0), 4)
    torch.cuda.current_stream().wait_stream(side)
    for n in ALL:
        assert torch.equal(want[n], got[n]), n


def test_graph_replays(gpu):
    """Forward and backward captured once and replayed on new inputs and lengths, with eager work between."""
    import flash_topk_attn_v2 as fta

    B, N, H, Hk, D = 2, 400, 4, 2, 128
    bufs = [torch.zeros_like(x) for x in _inputs(gpu, BF, B, N, H, Hk, D)]
    lens = torch.full((B,), N, dtype=torch.int32, device=gpu)
    q, k, v, do = bufs
    leaves = [x.requires_grad_(True) for x in (q, k, v)]

    def step():
        o, lse = fta.flash_window_attn(*leaves, H, (50, 0), 4, num_kv_heads=Hk, seq_lens=lens)
        return (o, lse, *torch.autograd.grad(o, leaves, do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, ln in enumerate(([400, 17], [3, 400], [256, 0])):
        new = _inputs(gpu, BF, B, N, H, Hk, D, seed=50 + 10 * i)
        with torch.no_grad():
            for x, y in zip(bufs, new):
                x.copy_(y)
            lens.copy_(torch.tensor(ln, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = dict(zip(ALL, (x.clone() for x in out)))
        want = _run(*new, H, Hk, (50, 0), 4, lens.clone())
        for n in ALL:
            assert torch.equal(want[n], got[n]), (i, n)


def test_gradient_by_differences(gpu):
    """dL along a direction against the change of L in float64 over a small step (the formula itself)."""
    q, k, v, do = _inputs(gpu, BF, 1, 90, 2, 1, 64)
    got = _run(q, k, v, do, 2, 1, (20, 4), 3)
    ins, h = [x.double() for x in (q, k, v)], 1e-4
    dirs = [torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).double().to(gpu) for i, x in enumerate(ins)]

    def loss(step):
        a, b, c = (x + step * d for x, d in zip(ins, dirs))
        o = 0.0
        for hd in range(2):
            r = R.attend(a[0].view(90, 2, 64)[:, hd], b[0], c[0], R.window_mask(90, 90, 0, 20, 4, 3, gpu), 1 / 8, BF)
            o = o + (r["o"] * do[0].view(90, 2, 64)[:, hd].double()).sum()
        return o

    slope = float((loss(h) - loss(-h)) / (2 * h))
    ref = R.window(q, k, v, 2, 1, 20, 4, 3, 1 / 8, None, do)
    along = sum(float((got[n].double() * d).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    tol = sum(float((ref[n + "_tol"] * d.abs()).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    exact = sum(float((ref[n] * d).sum()) for n, d in zip(("dq", "dk", "dv"), dirs))
    assert abs(exact - slope) <= 1e-5 * (1 + abs(slope))  # second-order term of a central difference at 1e-4
    assert abs(along - slope) <= tol + 1e-5 * (1 + abs(slope))


def test_unused_output_and_second_derivative(gpu):
    import flash_topk_attn_v2 as fta

    q, k, v, do = _inputs(gpu, BF, 1, 50, 2, 2, 64)
    q.requires_grad_(True)
    o, lse = fta.flash_window_attn(q, k, v, 2, (9, 0))
    assert o.requires_grad and not lse.requires_grad
    g, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    with torch.no_grad():
        o2, _ = fta.flash_window_attn(q, k, v, 2, (9, 0))
    assert not o2.requires_grad and torch.equal(o.detach(), o2)


def test_refusals(gpu):
    import flash_topk_attn_v2 as fta

    q, k = (torch.zeros(2, 5, n * 64, device=gpu, dtype=BF) for n in (4, 2))
    lens = torch.tensor([5, 3], dtype=torch.int32, device=gpu)
    good = dict(q=q, k=k, v=k, num_heads=4, window=(3, 0), num_kv_heads=2, seq_lens=lens)
    fta.flash_window_attn(**good)
    bad = [dict(q=q[0]), dict(q=q.float()), dict(v=k.half()), dict(k=k[:, :4]), dict(v=q), dict(num_heads=3), dict(num_kv_heads=4),
           dict(num_heads=32, num_kv_heads=16), dict(window=(-1, 0)), dict(window=(0, -2)), dict(window=(1, 2, 3)),
           dict(num_sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(seq_lens=lens.long()),
           dict(seq_lens=lens[:1]), dict(seq_lens=lens.cpu()), dict(k=k.cpu()), dict(q=q[:, :0], k=k[:, :0], v=k[:, :0])]
    for b in bad:
        with pytest.raises(ValueError):
            fta.flash_window_attn(**(good | b))


@pytest.mark.parametrize("case", range(12))
def test_drawn_shapes(gpu, case):
    """Shapes over the whole range, odd ones among them."""
    import random

    r = random.Random(case)
    dtype, D = r.choice([BF, FP]), r.choice([16, 64, 80, 128, 176, 256])
    Hk, G = r.choice([1, 2, 3]), r.choice([1, 2, 3, 4, 8])
    B, N = r.choice([1, 2, 3]), r.randrange(1, 900)
    left, right, sinks = r.randrange(0, 400), r.choice([0, 0, r.randrange(0, 300)]), r.choice([0, 1, 4, 33, 150])
    lens = [r.randrange(0, N + 1) for _ in range(B)] if r.random() < 0.5 else None
    say("window drawn", case, dtype, B, N, Hk * G, Hk, D, left, right, sinks, lens)
    q, k, v, do = _inputs(gpu, dtype, B, N, Hk * G, Hk, D, seed=1000 + case)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=gpu)
    got = _run(q, k, v, do, Hk * G, Hk, (left, right), sinks, ln)
    R.check(got, R.window(q, k, v, Hk * G, Hk, left, right, sinks, D ** -0.5, lens, do), ALL)
