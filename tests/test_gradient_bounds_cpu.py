"""That the gradient tests of the window attention can fail: mistakes planted in the float64 oracle leave
their bounds, without a GPU."""

import pytest
import torch

import _gradient_ref as G
import _operators_ref as R

ids = lambda c: "-".join(str(x) for x in c[1:9])  # noqa: E731


def _reference(case):
    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    q, k, v, do = G.inputs(case, "cpu")
    ref = R.window(q, k, v, H, Hk, left, right, sinks, D ** -0.5, lens, do)
    return (q, k, v, do), ref, ref["o"].to(dtype)


@pytest.mark.parametrize("case", G.CASES, ids=ids)
def test_a_wrong_delta_leaves_the_bounds(case):
    dtype, B, N, H, Hk, D, left, right, sinks, lens = case
    (q, k, v, do), ref, o = _reference(case)
    args = (q, k, v, o, do, H, Hk, left, right, sinks, D ** -0.5, lens)
    good = G.window(*args)
    for name in ("dq", "dk"):
        # the same formula as the other reference, up to what the rounded o moves
        assert ((good[name] - ref[name]).abs() <= ref[name + "_tol"]).all()
        assert (good[name + "_tol"] <= ref[name + "_tol"] * (1 + 1e-2)).all()
    for factor in (0.95, 1.05):
        bad = G.window(*args, delta_factor=factor)
        for name in ("dq", "dk"):
            off = (bad[name] - good[name]).abs() - good[name + "_tol"]  # less a rounding of the result
            assert (off > R.half_step(dtype) * good[name].abs()).any(), (name, factor)


@pytest.mark.parametrize("case", G.CASES, ids=ids)
def test_the_slope_is_far_larger_than_its_tolerance(case):
    (q, k, v, do), ref, _ = _reference(case)
    for name in ("dq", "dk", "dv"):
        d, slope, tol = G.along(case, q, k, v, do, ref, name)
        exact = float((ref[name] * d).sum())
        assert abs(exact - slope) <= 1e-6 * slope  # the formula itself; central differences in float64
        assert 0 < tol < slope / 3, (name, tol, slope)  # so that zeros, or two thirds of a gradient, fail
