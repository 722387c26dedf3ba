"""The passes along rows over more than 2^34 fp32 numbers, whose launches need more than one row of workgroups."""
import numpy as np
import pytest
import torch

import mx_ref as ref
from mx_gpu import assert_within, f64, values
from necklace_amd.cuda import mx

pytestmark = pytest.mark.gpu

ROWS, COLS = 131072 + 5, 131072  # 2^34 numbers and 5 rows: 2^32 lanes of 16 bytes are passed in the last ones
FIRST, LAST = [0, 1], [-2, -1]


def filled(x):
    """Zeros but for the first and the last two rows; those."""
    x.zero_()
    made = values(9, 4, COLS, torch.float32)
    x[FIRST], x[LAST] = made[:2], made[2:]
    return f64(made)


def ends(t):
    return torch.cat([t[:2], t[-2:]]).cpu().numpy()


def zero_between(t):
    return not bool(t[2:-2].any())


def test_passes_over_more_than_two_to_the_34_numbers():
    x = torch.empty(ROWS, COLS, device="cuda")
    v = filled(x)
    # 8 bits: save with an activation in place, load, gradient in place
    c, s = mx.act8_empty(ROWS, COLS)
    mx.cu_fn_act8_save_e(x, c, s, Y=x, fn="silu")
    wc, ws = ref.act8_quantize(v)
    assert np.array_equal(ends(c), wc) and np.array_equal(ends(s), ws) and zero_between(c) and zero_between(s)
    want = ref.activation(v, "silu")
    assert_within(ends(x).astype(np.float64), want, 2.0 ** -20 * np.abs(want) + 1e-30)
    assert zero_between(x)
    mx.cu_fn_act8_load_e(x, c, s)
    saved = ref.act8_decode(wc, ws, COLS)
    assert np.array_equal(ends(x), saved) and zero_between(x)
    x.fill_(1)
    mx.cu_fn_act8_grad_e(x, x, c, s, "silu")
    g = 1 / (1 + np.exp(-saved))
    want = g * (1 + saved * (1 - g))
    assert_within(ends(x).astype(np.float64), want, 2.0 ** -20 * (1 + np.abs(saved)))
    assert bool((x[2:-2] == 0.5).all())
    del c, s
    # 4 bits
    filled(x)
    c, s = mx.mx4_empty(ROWS, COLS)
    mx.cu_fn_mx4_quantize_e(x, c, s)
    wc, ws = ref.mx4_quantize(v)
    assert np.array_equal(ends(c), wc) and np.array_equal(ends(s), ws) and zero_between(c)
    x.fill_(1)
    mx.cu_fn_mx4_dequantize_e(x, c, s)
    assert np.array_equal(ends(x), ref.mx4_decode(wc, ws, COLS)) and zero_between(x)
    del x, c, s
    torch.cuda.empty_cache()
