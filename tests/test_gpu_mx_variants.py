"""Every kernel variant of the microscaled products, the weight gradient and the transposed quantise in its steady
state: many stages of the contracted length, odd and even, with ragged edges on every side.

Operands are quantised and decoded on the GPU (those passes are compared with numpy bit for bit elsewhere); results are
compared with products in 64 bits."""
import numpy as np
import pytest
import torch

from mx_gpu import DTYPES, half_step, name
from necklace_amd.cuda import mx

pytestmark = pytest.mark.gpu

PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def mx4_operand(g, rows, k, scale=1.0):
    """Codes, scales and the values they stand for in 64 bits."""
    c, s = mx.mx4_empty(rows, k)
    mx.cu_fn_mx4_quantize_e(torch.randn(rows, k, device="cuda", generator=g) * scale, c, s)
    v = torch.empty(rows, k, device="cuda")
    mx.cu_fn_mx4_dequantize_e(v, c, s)
    return c, s, v.double()


def act8_operand(g, t, k):
    x = torch.randn(t, k, device="cuda", generator=g)
    c, s = mx.act8_empty(t, k)
    mx.cu_fn_act8_save_e(x, c, s)
    mx.cu_fn_act8_load_e(x, c, s)
    return c, s, x.double()


def beyond(got, want, bound):
    off = (got.double() - want).abs() - bound
    return int((~(off <= 0)).sum())  # a NaN counts


# ---- products.  The bound of a result as in test_gpu_mx4: (128 + k / 64 + 8) * 2^-23 of the sum of magnitudes for the
# sums, one rounding to the type, half of fp16's smallest number.

def product_bound(a, bt, want, k, dtype):
    r = (128 + k / 64 + 8) * 2.0 ** -23 * (a.abs() @ bt.abs())
    return r + half_step(dtype) * (want.abs() + r) + (2.0 ** -25 if dtype == torch.float16 else 0)


# rows of 32 x 32; tiles 64 x 32, 64 x 64, 128 with four buffers, 128 with two, 256
OUTPUTS = [(17, 4000), (31, 3501), (37, 4100), (64, 3301), (1001, 1023), (1800, 2000), (2040, 2100), (3600, 3585)]


@pytest.mark.parametrize("k", [1030, 2100, 2300, 4100], ids=["9_steps", "17_steps", "18_steps", "33_steps"])
@pytest.mark.parametrize("m,n", OUTPUTS)
def test_products_of_many_steps(m, n, k):
    g = generator(m + k)
    ca, sa, a = mx4_operand(g, m, k)
    cb, sb, b = mx4_operand(g, n, k, 0.05)
    bt = b.t().contiguous()
    want = a @ bt
    dtype = DTYPES[(m + k) % 3]
    wide = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")
    y = wide[:, 1:1 + n]
    mx.cu_fn_mx4_matmul_e(y, ca, sa, cb, sb)
    assert beyond(y, want, product_bound(a, bt, want, k, dtype)) == 0
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + n:] == 7).all())
    # a block of NaN stays in its row of a, of b, whichever step it is in
    steps = mx.steps_of(k)
    rows, cols = [0, m // 2, m - 1], [5, n - 1]
    for i, row in enumerate(rows):
        sa[row, (4 * i * steps // len(rows)) + i] = 255
    sb[cols[0], 4 * (steps - 1)] = 255
    sb[cols[1], 4 * (steps // 2) + 3] = 255
    z = torch.empty(m, n, dtype=dtype, device="cuda")
    mx.cu_fn_mx4_matmul_e(z, ca, sa, cb, sb)
    assert bool(torch.isnan(z[rows]).all()) and bool(torch.isnan(z[:, cols]).all())
    z[rows] = y[rows]
    z[:, cols] = y[:, cols]
    assert torch.equal(z, y)


@pytest.mark.parametrize("m", [17, 24, 32, 33, 48, 64])
def test_linear_of_17_to_64_rows_against_thousands_of_columns(m):
    n, k = 4001, 2049
    g = generator(m)
    cb, sb, b = mx4_operand(g, n, k, 0.05)
    x = torch.randn(m, k, device="cuda", generator=g).to(torch.float16)
    bias = torch.randn(n, device="cuda", generator=g).to(torch.float16)
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    mx.cu_fn_mx4_linear_e(y, x, cb, sb, bias=bias)
    ca, sa = mx.mx4_empty(m, k)
    mx.cu_fn_mx4_quantize_e(x, ca, sa)
    a = torch.empty(m, k, device="cuda")
    mx.cu_fn_mx4_dequantize_e(a, ca, sa)
    a, bt = a.double(), b.t().contiguous()
    want = a @ bt + bias.double()
    bound = product_bound(a, bt, want, k, torch.float16) + 2.0 ** -24 * (a.abs() @ bt.abs() + bias.double().abs()) * (1 + 2.0 ** -11)
    assert beyond(y, want, bound) == 0


@pytest.mark.parametrize("dtype,rows,cols", [(torch.float32, 8191, 4097), (torch.bfloat16, 8191, 8201), (torch.float16, 8200, 8193)],
                         ids=["float32", "bfloat16", "float16"])
def test_transposed_codes_of_a_large_matrix(dtype, rows, cols):
    """The transposed quantise with 8 bytes a lane gives the codes of the transposed copy, bit for bit."""
    x = torch.randn(rows, cols, device="cuda", generator=generator(rows)).to(dtype)
    x[:, ::17] *= 20
    x[7, 5], x[rows - 1, cols - 1] = float("nan"), float("inf")
    c, s = mx.mx4_empty(cols, rows)
    mx.cu_fn_mx4_quantize_e(x, c, s, transpose=True)
    wc, ws = mx.mx4_empty(cols, rows)
    mx.cu_fn_mx4_quantize_e(x.t().contiguous(), wc, ws)
    assert torch.equal(c, wc) and torch.equal(s, ws)


# ---- weight gradient.  Bounds as in test_gpu_act8: (16 + parts * t / 16 + 257) * 2^-23 of the sum of magnitudes, db
# (t / 4 + 16 + 257) * 2^-24 of it.

# tiles of 256 cut in many parts, whole with few stages (13 of bf16, 25 of the others) and 272 tiles; of 128 whole; bf16
# 64 and the others 128 in 2 parts
WGRADS = [(11000, 1030, 1100), (777, 4000, 4000), (1000, 4096, 4300), (300, 1800, 2000), (2000, 1090, 1100)]


@pytest.mark.parametrize("t,n,k", WGRADS)
@pytest.mark.parametrize("odd", [0, 1], ids=["even_start", "odd_start"])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_weight_gradient(t, n, k, odd, dtype):
    """bf16 gradients at an even start go to LDS as they lie in memory, at an odd one through registers."""
    g = generator(t + n)
    c, s, x = act8_operand(g, t, k)
    wide = torch.full((t, n + 6), float("nan"), dtype=dtype, device="cuda")
    dy = wide[:, 2 + odd:2 + odd + n]
    dy.copy_(torch.randn(t, n, device="cuda", generator=g))
    area = torch.full((n, k + 5), 7.0, device="cuda")
    dw, db = area[:, 2:2 + k], torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d = dy.double().t().contiguous()
    want = d @ x
    bound = (16 + PARTS[dtype] * t / 16 + 257) * 2.0 ** -23 * (d.abs() @ x.abs())
    assert beyond(dw, want, bound) == 0
    want_b = d.sum(1)
    bound_b = (t / 4 + 16 + 257) * 2.0 ** -24 * d.abs().sum(1)
    assert beyond(db, want_b, bound_b) == 0
    assert bool((area[:, :2] == 7).all()) and bool((area[:, 2 + k:] == 7).all())
    again, again_b = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(again, dy, c, s)
    assert torch.equal(again, dw)
    again_b.copy_(db)
    mx.cu_fn_act8_wgrad_e(again, dy, c, s, DB=again_b, accumulate=True)
    assert beyond(again, 2 * want, 2 * bound + 2.0 ** -23 * want.abs()) == 0
    assert beyond(again_b, 2 * want_b, 2 * bound_b + 2.0 ** -23 * want_b.abs()) == 0


def one_token_a_column(t, n, dtype, g):
    """dy with one number a column, its token in every place of a stage in turn, with all bits of its type."""
    dy = torch.zeros(t, n, dtype=dtype, device="cuda")
    v = torch.randn(n, device="cuda", generator=g)
    v = torch.where(v.abs() < 2.0 ** -6, torch.ones_like(v) / 3, v).to(dtype)
    token = (torch.arange(n, device="cuda") * 37 + 5) % t
    dy[token, torch.arange(n, device="cuda")] = v
    return dy, token, v


@pytest.mark.parametrize("t,n,k", WGRADS + [(3000, 258, 32900), (60, 70, 90)])
@pytest.mark.parametrize("odd", [0, 1], ids=["even_start", "odd_start"])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_weight_gradient_keeps_every_bit(t, n, k, odd, dtype):
    """One product a result, of a number with all bits of its type and a power of two: nothing to round."""
    g = generator(n)
    x = torch.exp2(torch.randint(-3, 4, (t, k), device="cuda", generator=g).float())
    x *= torch.where(torch.rand(t, k, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    c, s = mx.act8_empty(t, k)
    mx.cu_fn_act8_save_e(x, c, s)
    made, token, v = one_token_a_column(t, n, dtype, g)
    wide = torch.empty(t, n + 2 + odd, dtype=dtype, device="cuda")
    dy = wide[:, odd:odd + n]
    dy.copy_(made)
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    assert torch.equal(dw, v.float().unsqueeze(1) * x[token])
    assert torch.equal(db, v.float())


@pytest.mark.parametrize("t,n,k", WGRADS)
@pytest.mark.parametrize("odd", [0, 1], ids=["even_start", "odd_start"])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_weight_gradient_with_nan_and_infinity(t, n, k, odd, dtype):
    """A NaN or an infinity reaches the results of its row and column and no other, in the first token, the last one and
    one between."""
    g = generator(k)
    x = torch.ones(t, k, device="cuda")
    x[0, 64:96] = float("nan")
    c, s = mx.act8_empty(t, k)
    mx.cu_fn_act8_save_e(x, c, s)
    wide = torch.empty(t, n + 2 + odd, dtype=dtype, device="cuda")
    dy = wide[:, odd:odd + n]
    dy.copy_(torch.randn(t, n, device="cuda", generator=g))
    dy[0, n - 1], dy[t - 1, 0], dy[t // 2, n // 2] = float("nan"), float("inf"), -float("inf")
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    fine = torch.ones(k, dtype=torch.bool, device="cuda")
    fine[64:96] = False
    assert bool(torch.isnan(dw[:, ~fine]).all())
    assert bool(torch.isnan(dw[n - 1]).all()) and bool(torch.isnan(db[n - 1]))
    assert bool((dw[0, fine] == np.inf).all()) and float(db[0]) == np.inf
    assert bool((dw[n // 2, fine] == -np.inf).all()) and float(db[n // 2]) == -np.inf
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[[0, n // 2, n - 1]] = False
    assert bool(torch.isfinite(dw[rest][:, fine]).all()) and bool(torch.isfinite(db[rest]).all())
