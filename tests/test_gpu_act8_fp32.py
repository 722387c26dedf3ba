"""fp32 activations and their slopes to a few roundings of the result, from tiny inputs to the tails.

Bounds in units of 2^-24, half a step of fp32 relative to the value (an instruction's 1 ulp counts as 2).
"""
import numpy as np
import pytest
import torch

import mx_ref as ref
from mx_gpu import assert_within, f64, packed8
from necklace_amd.cuda import mx

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24
NEAR = 1.25  # from here on gelu's smaller side is taken as e^(-x^2 / 2) times a polynomial
TINY = 2.0 ** -125  # what an instruction that flushes subnormal numbers may lose

RANGES = {"tiny": (-1e-6, 1e-6), "small": (-0.03, 0.03), "unit": (-3, 3), "border": (-1.3, -1.2), "negative": (-3, -1.25),
          "tail": (-6, -3), "far_tail": (-12, -6), "wide": (-60, 60)}


def inputs(which):
    lo, hi = RANGES[which]
    g = np.random.default_rng(len(which))
    return torch.from_numpy(g.uniform(lo, hi, (64, 512)).astype(np.float32)).cuda()


def side(x):
    """The smaller side of the normal distribution and the density."""
    return ref._normal(-np.abs(x)), np.exp(-x * x / 2) / np.sqrt(2 * np.pi)


# gelu.  |x| < 1.25: y = x^2 P(x^2) + x / 2 with one rounding of the sum; x^2 is rounded and |P| < 0.4; P's six terms
# have magnitudes that sum to 0.54 and two roundings each (the coefficient's and Horner's); the fit is off by
# 0.07 / 2 of |x|.  Beyond: y = max(x, 0) - |x| side with one rounding; side = t Q(t) e^(-x^2 / 2): t is off by 3 (the
# reciprocal 2, its argument 1), which t Q(t) carries on by the power 2.6 at most; Q's terms sum to 1.1 of Q with two
# roundings each; two products, the fit's 0.13; the exponential 2 and its argument, of x^2 / 2, 3 roundings.
def gelu_bound(x, y):
    a = np.abs(x)
    near = 1.5 * x * x + 0.04 * a + np.abs(y)
    s, _ = side(x)
    far = a * s * (14.2 + 1.5 * x * x) + np.abs(y)
    return np.where(a < NEAR, near, far) * HALF + TINY


# Its slope.  Near: x S(x^2) + 1/2 with one rounding; S's terms sum to 1.41 with two roundings each, the rounding of x^2
# moves S by 0.42, the fit is off by 0.013.  Far: w = e (t Q - |x| phi(0)) with e = e^(-x^2 / 2) (2 + 3 x^2 / 2 roundings),
# t Q off by 11.2, the constant and the sum by a rounding each, the product by one; w or 1 - w.
def gelu_slope_bound(x, want):
    a = np.abs(x)
    near = 3.3 * a + np.abs(want)
    s, d = side(x)
    far = 11.2 * s + a * d + (4 + 1.5 * x * x) * np.abs(s - a * d) + np.abs(want)
    return np.where(a < NEAR, near, far) * HALF + TINY


@pytest.mark.parametrize("which", RANGES)
def test_gelu(which):
    x = inputs(which)
    c, s = mx.act8_empty(*x.shape)
    y = torch.empty_like(x)
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn="gelu")
    want = ref.activation(f64(x), "gelu")
    assert_within(y, want, gelu_bound(f64(x), want))


@pytest.mark.parametrize("which", RANGES)
def test_gelu_slope(which):
    c, s, x = packed8(inputs(which))
    dx = torch.empty(x.shape, device="cuda")
    mx.cu_fn_act8_grad_e(dx, torch.full_like(dx, 2.0), c, s, "gelu")
    want = 2 * ref.slope(x, "gelu")
    assert_within(dx, want, 2 * gelu_slope_bound(x, want / 2))


@pytest.mark.parametrize("fn", ["gelu", "silu"])
def test_large_numbers_and_infinities(fn):
    big = float(np.finfo(np.float32).max)
    x = torch.tensor([[0.0, -0.0, 1e4, -1e4, 1e30, -1e30, big, -big, 13.3, -13.3, 14.6, -200.0]], device="cuda")
    c, s = mx.act8_empty(1, 12)
    y = torch.empty_like(x)
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn=fn)
    got = f64(y)[0]
    assert np.array_equal(got[[2, 4, 6]], f64(x)[0][[2, 4, 6]])
    assert np.all(np.abs(got[[0, 1, 3, 5, 7, 11]]) <= TINY)
    x[0, 4], x[0, 5], x[0, 8] = np.inf, -np.inf, np.nan
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn=fn)
    got = f64(y)[0]
    assert got[4] == np.inf and np.isnan(got[[5, 8]]).all()
    assert np.array_equal(got[[2, 6]], f64(x)[0][[2, 6]]) and np.all(np.abs(got[[0, 1, 3, 7, 11]]) <= TINY)
    # slopes of checkpoints of large numbers: 1 and 0
    for value, want in ((big, 1.0), (-big, 0.0), (1e20, 1.0), (-1e20, 0.0)):
        c, s, _ = packed8(torch.full((1, 12), value))
        dx = torch.empty(1, 12, device="cuda")
        mx.cu_fn_act8_grad_e(dx, torch.ones_like(dx), c, s, fn)
        assert bool((dx == want).all())


# silu.  x g with g = 1 / (1 + e) or e / (1 + e), e = e^-|x| off by the exponential's 2; sums, reciprocal and products are
# carried in two parts, whose own roundings are 2^-24 of 2^-24; the last sum 1.  Below x = -87 e may be flushed.
SILU_TINY = 2.0 ** -118


@pytest.mark.parametrize("which", RANGES)
def test_silu(which):
    x = inputs(which)
    c, s = mx.act8_empty(*x.shape)
    y = torch.empty_like(x)
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn="silu")
    want = ref.activation(f64(x), "silu")
    assert_within(y, want, 3.5 * HALF * np.abs(want) + SILU_TINY)


# g (1 + x h) with g and h = 1 - g off by 2 as above, two roundings of the sum, one of the product.
@pytest.mark.parametrize("which", RANGES)
def test_silu_slope(which):
    c, s, x = packed8(inputs(which))
    dx = torch.empty(x.shape, device="cuda")
    mx.cu_fn_act8_grad_e(dx, torch.full_like(dx, 2.0), c, s, "silu")
    g, h = 1 / (1 + np.exp(-x)), 1 / (1 + np.exp(x))
    want = g * (1 + x * h)
    assert_within(dx, 2 * want, 2 * HALF * (5.5 * np.abs(want) + 2.5 * g * h * np.abs(x)) + SILU_TINY)
