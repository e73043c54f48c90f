"""Norm and rotation of queries and keys, forward, backward and with the cache append,
against their definition in float64.

Bounds: every value is formed in fp32 from 16-bit inputs and rounded once, so an output
is off by u of its value plus fp32 errors, which are within 2^-18 of its terms'
magnitudes (sums of at most 256 squares, a dozen operations).  A weight gradient is a
sum of `rows` fp32 terms in fp32: (rows 2^-24 + 2^-18) of the terms' magnitudes at worst.
"""

import pytest
import torch

import _operators_ref as R
from _helpers import rand, say

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
F = 2.0 ** -18


def _tables(P, Rc, dev):
    inv = 10000.0 ** (-torch.arange(0, Rc, 2, dtype=torch.float64) / Rc)
    a = torch.arange(P, dtype=torch.float64)[:, None] * inv
    return a.cos().float().to(dev), a.sin().float().to(dev)


def _weight(D, seed, dtype, dev):
    return (1 + 0.3 * rand((D,), seed, F32, dev)).to(dtype)


def _close(got, want, mag, dtype, what):
    tol = R.half_step(dtype) * want.abs() + F * mag + R.tiny(dtype)
    off = (got.double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert (off <= tol).all(), f"{what}: {float((off / tol).max()):.2f} times the bound"


# dtype, weights' type (None: no weights), B, N, H, Hk, D, R, interleaved, positions
CASES = [
    (BF, F32, 1, 1, 1, 1, 16, 16, False, None),
    (FP, FP, 1, 3, 2, 1, 32, 16, True, None),
    (BF, BF, 2, 5, 3, 1, 48, 32, False, "batch"),
    (FP, F32, 2, 130, 4, 4, 64, 64, False, "row"),
    (BF, F32, 3, 77, 12, 4, 80, 32, True, "batch"),
    (BF, None, 1, 33, 6, 2, 96, 96, False, "long"),
    (FP, F32, 2, 257, 8, 2, 128, 128, True, None),
    (BF, F32, 2, 1025, 32, 8, 128, 128, False, "batch"),
    (BF, FP, 1, 40, 5, 5, 144, 48, False, None),
    (FP, BF, 2, 100, 4, 2, 256, 256, False, "long"),
    (BF, F32, 1, 3000, 2, 1, 64, 32, False, None),
    (BF, F32, 1, 4200, 64, 8, 128, 128, False, None),  # 69 MB: streamed past the caches
    (FP, F32, 2, 2100, 32, 8, 256, 64, True, "row"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[2:]))
def test_forward_and_gradients(gpu, case):
    import flash_topk_attn_v2 as fta

    dtype, wt, B, N, H, Hk, D, Rc, inter, how = case
    say("prep", case)
    P = N + 50
    cos, sin = _tables(P, Rc, gpu)
    g = torch.Generator().manual_seed(1)
    pos = None
    if how:
        pos = torch.randint(-20, P + 20, (N,) if how == "row" else (B, N), generator=g)  # outside: the nearest row
        pos = pos.to(gpu, torch.int64 if how == "long" else torch.int32)
        if how == "long":
            pos[0, 0] = 1 << 40
    q, dq = (rand((B, N, H * D), i, dtype, gpu) for i in (2, 3))
    k, dk = (rand((B, N, Hk * D), i, dtype, gpu) for i in (4, 5))
    ws = [None if wt is None else _weight(D, 6 + i, wt, gpu) for i in range(2)]
    ins = [x if x is None else x.detach().requires_grad_(True) for x in (q, k, *ws)]
    out = fta.flash_qk_norm_rope(ins[0], ins[1], H, cos, sin, ins[2], ins[3], eps=1e-5, num_kv_heads=Hk, positions=pos,
                                 interleaved=inter)
    got = torch.autograd.grad(out, [x for x in ins if x is not None], (dq, dk))
    at = torch.arange(N, device=gpu).expand(B, N) if pos is None else pos.expand(B, N)
    for i, (x, d, heads, y) in enumerate(((q, dq, H, out[0]), (k, dk, Hk, out[1]))):
        x64 = x.double().requires_grad_(True)
        w64 = None if wt is None else ws[i].double().requires_grad_(True)
        ref = R.turned(x64, heads, w64, cos, sin, at, 1e-5, inter)
        mag = R.turned(x64.detach().abs(), heads, None if wt is None else w64.detach().abs(), cos.abs(), -sin.abs(), at,
                       1e-5, inter).abs() + 2 * R.turned(x64.detach().abs(), heads, None if wt is None else w64.detach().abs(),
                                                         cos.abs(), sin.abs(), at, 1e-5, inter).abs()
        _close(y.detach(), ref.detach(), mag, dtype, f"{case} y{i}")
        grads = torch.autograd.grad(ref, [x64] if wt is None else [x64, w64], d.double())
        # magnitude of dx's terms: r (|h| + |n| mean |h n|) with |h| <= |w| (|dy_a| + |dy_b|)
        xs, ds = (t.detach().double().view(B, N, heads, D) for t in (x, d))
        r = (xs.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        n = xs * r
        pair = torch.arange(D, device=gpu)
        turn = pair < Rc
        other = torch.where(turn, (pair ^ 1) if inter else (pair + Rc // 2) % Rc, pair)
        gm = ds.abs() + torch.where(turn, ds.abs()[..., other], 0.0)
        hm = gm * (1.0 if wt is None else ws[i].double().abs())
        mag = (r * (hm + n.abs() * (hm * n.abs()).mean(-1, keepdim=True))).flatten(-2)
        _close(got[i], grads[0], mag, dtype, f"{case} dx{i}")
        if wt is not None:
            terms = (gm * n.abs()).sum((0, 1, 2))
            tol = (B * N * heads * 2.0 ** -24 + F) * terms + (R.half_step(wt) * grads[1].abs())
            off = (got[2 + i].double() - grads[1]).abs()
            assert got[2 + i].dtype == wt and (off <= tol).all(), f"{case} dw{i}: {float((off / tol).max()):.2f}"


def test_only_some_gradients(gpu):
    """Frozen weights, one weight alone, one output unused."""
    import flash_topk_attn_v2 as fta

    q, k, dq = (rand((1, 9, 64), i, BF, gpu) for i in range(3))
    cos, sin = _tables(9, 32, gpu)
    qw, kw = _weight(32, 4, F32, gpu), _weight(32, 5, F32, gpu)
    qr, kr, qwr = (x.detach().requires_grad_(True) for x in (q, k, qw))
    a, b = fta.flash_qk_norm_rope(qr, kr, 2, cos, sin, qwr, kw)
    full = torch.autograd.grad((a, b), (qr, kr, qwr), (dq, torch.zeros_like(b)), retain_graph=True)
    part = torch.autograd.grad(a, (qr, kr, qwr), dq)
    for x, y in zip(full, part):
        assert torch.equal(x, y)
    assert (part[1] == 0).all()
    a2, _ = fta.flash_qk_norm_rope(qr, k, 2, cos, sin, qw, kw)
    assert torch.equal(torch.autograd.grad(a2, qr, dq)[0], full[0])
    a3, _ = fta.flash_qk_norm_rope(q, k, 2, cos, sin, qw, None)  # one weight of two
    assert torch.equal(a3, a.detach())


def test_layouts_streams_and_same_bits(gpu):
    import flash_topk_attn_v2 as fta

    packed = rand((2, 50, 6 * 64), 3, BF, gpu)
    q, k = packed[..., :256], packed[..., 256:]
    cos, sin = _tables(60, 64, gpu)
    w = _weight(64, 4, F32, gpu)
    want = fta.flash_qk_norm_rope(q.contiguous(), k.contiguous(), 4, cos, sin, w, w, num_kv_heads=2)
    wide = torch.zeros(60, 40, device=gpu)
    wide[:, 3:35] = cos  # a table that is a view, off the 16-byte grid
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fta.flash_qk_norm_rope(q, k, 4, wide[:, 3:35], sin, w, w, num_kv_heads=2)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(want, got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,B,T,H,Hk,D,Rc,S,inter,offset", [
    (BF, 1, 1, 8, 8, 64, 64, 40, False, 0), (FP, 5, 3, 4, 2, 128, 64, 64, True, 7), (BF, 130, 1, 32, 8, 128, 128, 33, False, 100),
    (FP, 4, 2, 3, 1, 80, 32, 9, False, 0), (BF, 2, 70, 4, 2, 256, 256, 100, False, 3),
    (BF, 130, 10, 32, 8, 128, 128, 33, False, 0)])
def test_append(gpu, dtype, B, T, H, Hk, D, Rc, S, inter, offset):
    import flash_topk_attn_v2 as fta

    say("append", dtype, B, T, H, Hk, D, Rc, S)
    q, k, v = rand((B, T, H * D), 1, dtype, gpu), rand((B, T, Hk * D), 2, dtype, gpu), rand((B, T, Hk * D), 3, dtype, gpu)
    kc, vc = rand((B, S, Hk * D), 4, dtype, gpu), rand((B, S, Hk * D), 5, dtype, gpu)
    cos, sin = _tables(S + offset, Rc, gpu)
    qw, kw = _weight(D, 6, F32, gpu), _weight(D, 7, F32, gpu)
    # ordinary lengths, then a request with fewer tokens than T, an idle one and one past the cache
    lens = torch.randint(T, S + 1, (B,), generator=torch.Generator().manual_seed(8)).int()
    lens[-3:] = torch.tensor([T - 1, 0, S + 1])[-min(B, 3):] if B > 1 else lens[-3:]
    lens = lens.to(gpu)
    k0, v0, ver = kc.clone(), vc.clone(), kc._version
    out = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos, sin, qw, kw, num_kv_heads=Hk,
                                        position_offset=offset, interleaved=inter)
    assert kc._version > ver
    row = lens.long()[:, None] - T + torch.arange(T, device=gpu)
    # the training operator on the same tokens: the same bits
    pos = (row + offset).int()
    wq, wk = fta.flash_qk_norm_rope(q, k, H, cos, sin, qw, kw, num_kv_heads=Hk, positions=pos, interleaved=inter)
    assert torch.equal(out, wq)
    for b in range(B):
        for t in range(T):
            r = int(row[b, t])
            if 0 <= r < S:
                k0[b, r], v0[b, r] = wk[b, t], v[b, t]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # every other row as it was


def test_append_into_views(gpu):
    """Caches that are one tensor's halves, head-major batches: only the rows that belong there change."""
    import flash_topk_attn_v2 as fta

    B, T, H, D, S = 3, 2, 2, 64, 11
    both = rand((S, B, 2 * H * D), 1, BF, gpu)
    kc, vc = both.transpose(0, 1).split(H * D, -1)
    q, k, v = (rand((B, T, H * D), i, BF, gpu) for i in (2, 3, 4))
    cos, sin = _tables(S, 64, gpu)
    lens = torch.tensor([2, 11, 7], dtype=torch.int32, device=gpu)
    kd, vd = kc.contiguous(), vc.contiguous()
    a = fta.flash_qk_norm_rope_append(q, k, v, kd, vd, lens, H, cos, sin)
    b = fta.flash_qk_norm_rope_append(q, k, v, kc, vc, lens, H, cos, sin)
    assert torch.equal(a, b) and torch.equal(kd, kc) and torch.equal(vd, vc)


def test_unaligned_addresses(gpu):
    """Contiguous tensors whose first element is off the 16-byte grid."""
    import flash_topk_attn_v2 as fta

    def shifted(x):
        y = torch.empty(x.numel() + 3, device=gpu, dtype=x.dtype)[3:].view(x.shape)
        return y.copy_(x)

    q, k = rand((2, 9, 128), 1, BF, gpu), rand((2, 9, 64), 2, BF, gpu)
    cos, sin = _tables(9, 32, gpu)
    w = _weight(64, 4, FP, gpu)
    want = fta.flash_qk_norm_rope(q, k, 2, cos, sin, w, w, num_kv_heads=1)
    got = fta.flash_qk_norm_rope(shifted(q), shifted(k), 2, shifted(cos), shifted(sin), shifted(w), w, num_kv_heads=1)
    for x, y in zip(want, got):
        assert torch.equal(x, y)
    kc = torch.zeros(2, 20, 64, device=gpu, dtype=BF)
    lens = torch.tensor([9, 20], dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError, match="16-byte aligned"):
        fta.flash_qk_norm_rope_append(q, k, k, shifted(kc), kc, lens, 2, cos, sin, num_kv_heads=1)


def test_modes(gpu):
    """Inference mode, a second derivative (refused) and calls that would lose a gradient (refused)."""
    import flash_topk_attn_v2 as fta

    cos, sin = _tables(8, 64, gpu)
    lens = torch.tensor([4], dtype=torch.int32, device=gpu)
    with torch.inference_mode():
        x = rand((1, 4, 64), 1, BF, gpu)
        c = torch.zeros(1, 8, 64, device=gpu, dtype=BF)
        out = fta.flash_qk_norm_rope_append(x, x, x, c, c.clone(), lens, 1, cos, sin)
        a, b = fta.flash_qk_norm_rope(x, x, 1, cos, sin)
        assert torch.equal(out, a) and torch.equal(c[:, :4], b)
    q = rand((1, 4, 64), 1, BF, gpu).requires_grad_(True)
    a, _ = fta.flash_qk_norm_rope(q, q.detach(), 1, cos, sin)
    g, = torch.autograd.grad(a.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    c = torch.zeros(1, 8, 64, device=gpu, dtype=BF)
    with pytest.raises(ValueError, match="not differentiable"):
        fta.flash_qk_norm_rope_append(q, q, q, c, c.clone(), lens, 1, cos, sin)


def test_refusals(gpu):
    import flash_topk_attn_v2 as fta

    q, k = (torch.zeros(2, 5, n * 64, device=gpu, dtype=BF) for n in (4, 2))
    cos, sin = _tables(6, 64, gpu)
    w = torch.ones(64, device=gpu)
    good = dict(q=q, k=k, num_heads=4, cos=cos, sin=sin, q_weight=w, k_weight=w, num_kv_heads=2)
    fta.flash_qk_norm_rope(**good)
    bad = [dict(q=q[0]), dict(q=q.float()), dict(k=k.half()), dict(k=k[:, :4]), dict(k=q), dict(num_heads=3), dict(num_heads=0),
           dict(num_kv_heads=3), dict(num_heads=32, num_kv_heads=16), dict(cos=cos[:4], sin=sin[:4]), dict(cos=cos[:, :3]),
           dict(cos=cos.half(), sin=sin.half()), dict(cos=cos[:, :4], sin=sin[:, :4]), dict(cos=cos.cpu()), dict(eps=0.0),
           dict(eps=float("nan")), dict(q_weight=w[:32]), dict(q_weight=w.half()), dict(q_weight=w.double(), k_weight=w.double()),
           dict(q_weight=w.cpu()), dict(cos=cos.clone().requires_grad_(True)),
           dict(positions=torch.zeros(2, 4, device=gpu, dtype=torch.int32)), dict(positions=torch.zeros(2, 5, device=gpu)),
           dict(positions=torch.zeros(2, 5, dtype=torch.int32)), dict(q=q[:0], k=k[:0])]
    for b in bad:
        with pytest.raises(ValueError):
            fta.flash_qk_norm_rope(**(good | b))
    kc, vc = (torch.zeros(2, 9, 128, device=gpu, dtype=BF) for _ in range(2))
    lens = torch.tensor([5, 9], dtype=torch.int32, device=gpu)
    good |= dict(v=k, k_cache=kc, v_cache=vc, cache_lens=lens)
    with torch.no_grad():
        fta.flash_qk_norm_rope_append(**good)
        bad = [dict(v=q), dict(v=k.half()), dict(k_cache=kc[:1]), dict(v_cache=vc[:, :8]), dict(k_cache=kc.half()),
               dict(cache_lens=lens.long()), dict(cache_lens=lens[:1]), dict(cache_lens=lens.cpu()),
               dict(k_cache=kc[:1].expand(2, -1, -1)), dict(v_cache=vc[:, :1].expand(-1, 9, -1)), dict(position_offset=1 << 40),
               dict(k_cache=torch.zeros(2, 9, 256, device=gpu, dtype=BF)[..., ::2]), dict(k_cache=kc[:, :0], v_cache=vc[:, :0])]
        for b in bad:
            with pytest.raises(ValueError):
                fta.flash_qk_norm_rope_append(**(good | b))
