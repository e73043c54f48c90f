"""Gradients of the window attention against differences along the gradient itself, and against the formula
with delta from the kernel's own output, in float64."""

import itertools

import pytest
import torch

import _gradient_ref as G
import _operators_ref as R
from _helpers import say

pytestmark = pytest.mark.gpu

ids = lambda c: "-".join(str(x) for x in c[1:9])  # noqa: E731


def _run(case, q, k, v, do, wanted=(True, True, True)):
    import flash_topk_attn_v2 as fta

    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    x = [t.detach().requires_grad_(w) for t, w in zip((q, k, v), wanted)]
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=q.device)
    o, _ = fta.flash_window_attn(*x, H, (left, right), sinks, num_kv_heads=Hk, seq_lens=ln)
    grads = iter(torch.autograd.grad(o, [t for t in x if t.requires_grad], do))
    return o.detach(), [next(grads) if w else None for w in wanted]


@pytest.mark.parametrize("case", G.CASES, ids=ids)
def test_gradients_with_delta_of_the_own_output(gpu, case):
    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    say("own delta", case)
    q, k, v, do = G.inputs(case, gpu)
    o, (dq, dk, _) = _run(case, q, k, v, do)
    ref = G.window(q, k, v, o, do, H, Hk, left, right, sinks, D ** -0.5, lens)
    R.check({"dq": dq, "dk": dk}, ref, ("dq", "dk"), str(case))


@pytest.mark.parametrize("case", G.CASES, ids=ids)
def test_slopes_along_the_gradients(gpu, case):
    """Each gradient alone, along itself: the slope is several times the worst error."""
    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    say("slopes", case)
    q, k, v, do = G.inputs(case, gpu)
    _, grads = _run(case, q, k, v, do)
    ref = R.window(q, k, v, H, Hk, left, right, sinks, D ** -0.5, lens, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        d, slope, tol = G.along(case, q, k, v, do, ref, name)
        got = float((got.double() * d).sum())
        assert abs(got - slope) <= tol + 1e-6 * slope, (name, got, slope, tol)


@pytest.mark.parametrize("case", G.CASES[:3] + G.CASES[6:7], ids=ids)
def test_some_gradients_are_the_full_ones(gpu, case):
    """Frozen inputs change no other gradient's bits."""
    q, k, v, do = G.inputs(case, gpu)
    _, full = _run(case, q, k, v, do)
    for wanted in itertools.product((True, False), repeat=3):
        if any(wanted):
            for w, x, y in zip(wanted, full, _run(case, q, k, v, do, wanted)[1]):
                assert not w or torch.equal(x, y), wanted


@pytest.mark.parametrize("dtype,B,N,H,Hk,D,left,right,sinks,lens", [
    (torch.bfloat16, 4, 200, 8, 8, 64, 1, 0, 0, None),       # two keys a row
    (torch.float16, 2, 200, 8, 4, 128, 3, 0, 1, [200, 77]),
    (torch.bfloat16, 2, 300, 4, 1, 256, 3, 4, 0, None),
    (torch.float16, 3, 300, 4, 4, 64, 20, 10, 2, None),
    (torch.bfloat16, 64, 16, 4, 2, 128, 100, 0, 0, None),    # causal, sixteen tokens
    (torch.bfloat16, 16, 63, 4, 2, 80, 100, 100, 0, None),   # everything of a few tokens
    (torch.float16, 40, 33, 3, 1, 160, 40, 0, 4, None),
    (torch.bfloat16, 64, 60, 4, 4, 64, 60, 0, 0, [2 + i % 7 for i in range(64)]),
])
def test_rows_that_see_few_keys(gpu, dtype, B, N, H, Hk, D, left, right, sinks, lens):
    """dQ and dK of rows that see few keys are as near as those of rows that see many.

    dS and the gradient are each rounded once to 16 bits, independently, so the gradient is off by sqrt(2)
    times what rounding the exact one costs; 1.5 leaves 6% for the sample.  delta from the rounded o
    would be 1.6 times (8 keys) to 2.3 (2 keys).
    """
    say("few keys", dtype, B, N, H, Hk, D, left, right, sinks)
    case = (dtype, B, N, H, Hk, D, left, right, sinks, lens)
    q, k, v, do = G.inputs(case, gpu)
    _, grads = _run(case, q, k, v, do)
    ref = R.window(q, k, v, H, Hk, left, right, sinks, D ** -0.5, lens, do)
    for name, got in zip(("dq", "dk", "dv"), grads):
        want = ref[name]
        rounding = (want.to(dtype).double() - want).norm()
        off = (got.double() - want).norm()
        assert off <= 1.5 * rounding, (name, float(off / rounding))
    R.check(dict(zip(("dq", "dk", "dv"), grads)), ref, ("dq", "dk", "dv"))


@pytest.mark.parametrize("dtype,N,D,left,right", [(torch.float16, 40000, 64, 40000, 40000), (torch.float16, 70000, 128, 70000, 0),
                                                  (torch.float16, 33000, 256, 33000, 33000), (torch.bfloat16, 33000, 64, 33000, 0)])
def test_long_sequences_keep_small_probabilities(gpu, dtype, N, D, left, right):
    """dV where every probability is below fp16's normal range (the mean is 1 / N).

    P and dV are each rounded once, independently: sqrt(2) times what rounding the exact dV costs, and 6%
    for the sample.  P in fp16 as it stands would be 2.1 (32768 keys) to 6.5 times (131072).
    """
    say("long", dtype, N, D, left, right)
    q, k, v, do = G.inputs((dtype, 1, N, 1, 1, D), gpu)
    _, (_, _, dv) = _run((dtype, 1, N, 1, 1, D, left, right, 0, None), q, k, v, do)
    want = torch.zeros(N, D, device=gpu, dtype=torch.float64)
    kd, j = k[0].double(), torch.arange(N, device=gpu)
    for i in range(0, N, 1024):
        rows = torch.arange(i, min(N, i + 1024), device=gpu)[:, None]
        s = (q[0, i:i + 1024].double() @ kd.T * D ** -0.5).masked_fill_((j > rows + right) | (j < rows - left), -float("inf"))
        want += torch.softmax(s, -1).T @ do[0, i:i + 1024].double()
    off, rounding = (dv[0].double() - want).norm(), (want.to(dtype).double() - want).norm()
    assert off <= 1.5 * rounding, float(off / rounding)
