"""mx4 quantise, decode, product and linear against the numpy reference in 64 bits."""
import numpy as np
import pytest
import torch

import mx_ref as ref
from mx_gpu import DTYPES, assert_within, f64, half_step, matmul64, name, packed4, untouched, values, widened
from necklace_amd import _lib
from necklace_amd.cuda import mx

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 31), (1, 32), (3, 33), (7, 127), (5, 128), (4, 129), (33, 1000), (257, 64), (130, 517), (1, 5000),
          (1025, 96)]


def quantize(x, transpose=False):
    rows, cols = mx.shape2(x)
    if transpose:
        rows, cols = cols, rows
    c, s = mx.mx4_empty(rows, cols)
    c.fill_(0xAA)
    s.fill_(0xAA)
    mx.cu_fn_mx4_quantize_e(x, c, s, transpose=transpose)
    return c, s


def assert_codes(c, s, x64, what=""):
    wc, ws = ref.mx4_quantize(x64)
    assert np.array_equal(s.cpu().numpy(), ws), f"{what}: scales"
    assert np.array_equal(c.cpu().numpy(), wc), f"{what}: codes"


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "transpose"])
def test_codes_and_scales(rows, cols, dtype, transpose):
    x = values(rows * 7 + cols, rows, cols, dtype)
    c, s = quantize(x, transpose)
    assert_codes(c, s, f64(x).T if transpose else f64(x))


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "transpose"])
def test_ties_subnormals_and_non_finite_values(dtype, transpose):
    """Every middle between two codes and its neighbours at scales over the type's whole range; infinities and NaN."""
    t = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.5])
    fi = torch.finfo(dtype)
    low = int(np.floor(np.log2(fi.smallest_normal))) - (2 if dtype == torch.float16 else 6)
    top = int(np.floor(np.log2(fi.max))) - 2
    rows = []
    for e in sorted({low, low + 1, low + 3, -126, -125, -20, -1, 0, 1, 10, top} & set(range(low, top + 1))):
        base = t.double() * 2.0 ** e
        near = torch.cat([base, base * (1 + 2 * fi.eps), base * (1 - fi.eps)])
        near = torch.cat([near, -near])
        near = near[near.abs() < fi.max]
        for start in range(0, near.numel(), 31):  # a largest value of 4 scales keeps the scale at 2^e
            part = torch.zeros(32, dtype=torch.float64)
            part[0] = 4 * 2.0 ** e
            chunk = near[start:start + 31]
            part[1:1 + chunk.numel()] = chunk
            rows.append(part)
    for bad in (float("inf"), -float("inf"), float("nan")):
        part = torch.ones(32, dtype=torch.float64)
        part[len(rows) % 32] = bad
        rows.append(part)
    rows.append(torch.full((32,), -0.0, dtype=torch.float64))
    x = torch.stack(rows).to(dtype).cuda()
    x = torch.cat([x, x.flip(0)], 1)
    c, s = quantize(x.t().contiguous() if transpose else x, transpose)
    assert_codes(c, s, f64(x))
    out = torch.zeros_like(x)
    mx.cu_fn_mx4_dequantize_e(out, c, s)
    want = ref.mx4_decode(c.cpu().numpy(), s.cpu().numpy(), x.shape[1])
    want = torch.from_numpy(want).to(dtype).double().numpy()  # rounds in fp16 only
    assert np.array_equal(f64(out), want, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_decode_any_codes(rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    steps = ref.steps_of(cols)
    c = rng.integers(0, 256, (rows, steps * 64), dtype=np.uint8)
    s = rng.integers(0, 256, (rows, steps * 4), dtype=np.uint8)
    s[0, 0] = 255
    want = ref.mx4_decode(c, s, cols)
    with np.errstate(over="ignore"):
        want = torch.from_numpy(want).to(torch.float32).to(dtype).double().numpy()
    out, wide = widened(torch.zeros(rows, cols, dtype=dtype, device="cuda"))
    mx.cu_fn_mx4_dequantize_e(out, torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda())
    assert np.array_equal(f64(out), want, equal_nan=True)
    assert untouched(wide, 3, cols)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "transpose"])
@pytest.mark.parametrize("left", [1, 2, 8])
def test_column_ranges_and_odd_starts(dtype, transpose, left):
    x = values(5, 70, 300, dtype)
    view, _ = widened(x, left, 6)
    assert_codes(*quantize(view, transpose), f64(x).T if transpose else f64(x))


def test_more_dimensions_and_vectors():
    x = values(1, 6 * 5, 40, torch.bfloat16)
    c, s = mx.mx4_empty(30, 40)
    mx.cu_fn_mx4_quantize_e(x.view(2, 3, 5, 40), c, s)
    assert_codes(c, s, f64(x))
    c, s = mx.mx4_empty(1, 40)
    mx.cu_fn_mx4_quantize_e(x[3], c, s)
    assert_codes(c, s, f64(x)[3:4])


# ---- products.  Every product of two values is exact; an instruction sums 64 or 128 of them, so a result carries at
# most that many roundings of its own partial sums, one more for every further step of k, 8 for joining waves: at
# most (128 + k / 64 + 8) * 2^-23 of the sum of magnitudes (2^-23: truncation as well as rounding is covered), one
# rounding for the bias and one to the output type.

def product_bound(a, b, want, k, dtype, bias=None):
    mags = matmul64(np.abs(a), np.abs(b).T)
    r = (128 + k / 64 + 8) * 2.0 ** -23 * mags
    if bias is not None:
        r = r + 2.0 ** -24 * (mags + np.abs(bias))
    return r + half_step(dtype) * (np.abs(want) + r) + (2.0 ** -25 if dtype == torch.float16 else 0)


PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 1024, 1024), (3, 17, 100), (8, 40, 2050), (9, 33, 129), (16, 100, 4096), (17, 50, 300),
            (37, 96, 1500), (64, 65, 257), (65, 64, 128), (100, 130, 640), (129, 257, 1000), (1000, 500, 384),
            (700, 2500, 129), (1800, 2000, 260), (3600, 3585, 257)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype,with_bias", [(torch.float32, True), (torch.bfloat16, False), (torch.float16, True)],
                         ids=["float32_bias", "bfloat16", "float16_bias"])
def test_product(m, n, k, dtype, with_bias):
    ca, sa, a = packed4(f64(values(m, m, k, torch.float32)))
    cb, sb, b = packed4(f64(values(n + 1, n, k, torch.float32, 0.05)))
    bias = torch.linspace(-2, 2, n).to(dtype).cuda() if with_bias else None
    want = matmul64(a, b.T) + (f64(bias) if with_bias else 0)
    bound = product_bound(a, b, want, k, dtype, f64(bias) if with_bias else None)
    y, wide = widened(torch.zeros(m, n, dtype=dtype, device="cuda"))
    mx.cu_fn_mx4_matmul_e(y, ca, sa, cb, sb, bias=bias)
    assert_within(y, want, bound, "matmul")
    assert untouched(wide, 3, n)


@pytest.mark.parametrize("m,n,k", [p for p in PRODUCTS if p[0] <= 1000] + [(5, 20, 33), (8, 8, 1023), (2, 70, 8191)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_linear_is_quantise_and_product(m, n, k, dtype):
    """The same bits as the two calls, which the tests above compare with the definition."""
    x, _ = widened(values(m + 2, m, k, dtype), 1, 2)
    cb, sb, _ = packed4(f64(values(n + 1, n, k, torch.float32, 0.05)))
    bias = torch.linspace(-1, 1, n).to(dtype).cuda()
    y, wide = widened(torch.zeros(m, n, dtype=dtype, device="cuda"))
    mx.cu_fn_mx4_linear_e(y, x, cb, sb, bias=bias)
    ca, sa = quantize(x)
    z = torch.empty(m, n, dtype=dtype, device="cuda")
    mx.cu_fn_mx4_matmul_e(z, ca, sa, cb, sb, bias=bias)
    assert torch.equal(y, z)
    assert untouched(wide, 3, n)


@pytest.mark.parametrize("m", [1, 8, 20, 200])
def test_an_input_row_with_nan_or_infinity_stays_in_its_row(m):
    x = values(3, m, 256, torch.bfloat16)
    x[m - 1, 200] = float("nan")
    if m > 1:
        x[0, 7] = float("inf")
    cb, sb, _ = packed4(f64(values(4, 48, 256, torch.float32)))
    y = torch.zeros(m, 48, dtype=torch.bfloat16, device="cuda")
    mx.cu_fn_mx4_linear_e(y, x, cb, sb)
    assert torch.isnan(y[m - 1]).all() and torch.isnan(y[0]).all()
    assert torch.isfinite(y[1:m - 1]).all()


@pytest.mark.parametrize("m", [1, 3, 100])
def test_no_columns_give_the_bias(m):
    ca, sa = mx.mx4_empty(m, 0)
    cb, sb = mx.mx4_empty(5, 0)
    bias = torch.arange(5.0, device="cuda")
    y = torch.full((m, 5), 7.0, device="cuda")
    mx.cu_fn_mx4_matmul_e(y, ca, sa, cb, sb, bias=bias)
    assert torch.equal(y, bias.expand(m, 5))
    y.fill_(7)
    mx.cu_fn_mx4_linear_e(y, torch.empty(m, 0, device="cuda"), cb, sb)
    assert not y.any()


def test_empty_outputs():
    c, s = mx.mx4_empty(4, 64)
    none_c, none_s = mx.mx4_empty(0, 64)
    mx.cu_fn_mx4_quantize_e(torch.empty(0, 64, device="cuda"), none_c, none_s)
    mx.cu_fn_mx4_matmul_e(torch.empty(0, 4, device="cuda"), none_c, none_s, c, s)
    mx.cu_fn_mx4_linear_e(torch.empty(4, 0, device="cuda"), torch.empty(4, 64, device="cuda"), none_c, none_s)


def test_gradient_of_a_product_through_the_transpose():
    """d/dx of sum(dy * x W^T) is dy W: through codes of W^T, against the formula of the decoded codes."""
    dy = values(1, 50, 70, torch.float32)
    w = values(2, 70, 90, torch.float32)
    ct, st = quantize(w, transpose=True)
    dx = torch.empty(50, 90, device="cuda")
    mx.cu_fn_mx4_linear_e(dx, dy, ct, st)
    a = ref.mx4_decode(*ref.mx4_quantize(f64(dy)), 70)
    b = ref.mx4_decode(*ref.mx4_quantize(f64(w).T), 70)
    want = matmul64(a, b.T)
    assert_within(dx, want, product_bound(a, b, want, 70, torch.float32))


def test_refusals_of_tensors_that_do_not_fit():
    x = torch.zeros(4, 300, device="cuda")
    c, s = mx.mx4_empty(4, 300)
    with pytest.raises(ValueError, match="does not match"):
        mx.cu_fn_mx4_quantize_e(x[:3], c, s)
    with pytest.raises(ValueError, match="does not match"):
        mx.cu_fn_mx4_quantize_e(x, c, s, transpose=True)
    with pytest.raises(ValueError, match="scales of C"):
        mx.cu_fn_mx4_quantize_e(x, c, s[:, :4])
    with pytest.raises(ValueError, match="neighbouring"):
        mx.cu_fn_mx4_quantize_e(x.t(), *mx.mx4_empty(300, 4))
    with pytest.raises(ValueError, match="neighbouring"):
        mx.cu_fn_mx4_quantize_e(x[:1].expand(4, 300), c, s)
    with pytest.raises(TypeError, match="uint8"):
        mx.cu_fn_mx4_dequantize_e(x, c.view(torch.int8), s)
    with pytest.raises(ValueError, match="contiguous"):
        wide = torch.zeros(4, 400, dtype=torch.uint8, device="cuda")
        mx.cu_fn_mx4_dequantize_e(x, wide[:, :192], s)
    y = torch.zeros(4, 4, device="cuda")
    with pytest.raises(ValueError, match="CB"):
        mx.cu_fn_mx4_matmul_e(y, c, s, *mx.mx4_empty(4, 500))
    with pytest.raises(TypeError, match="X is"):
        mx.cu_fn_mx4_linear_e(y, x.bfloat16(), c, s)
    with pytest.raises(ValueError, match="rows"):
        mx.cu_fn_mx4_linear_e(y, x[:2], c, s)
    with pytest.raises(ValueError, match="bias"):
        mx.cu_fn_mx4_linear_e(y, x, c, s, bias=torch.zeros(5, device="cuda"))
    with pytest.raises(TypeError, match="bias"):
        mx.cu_fn_mx4_linear_e(y, x, c, s, bias=torch.zeros(4, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="workspace"):
        mx.cu_fn_mx4_linear_e(y, x, c, s, workspace=torch.zeros(4, device="cuda"))
    big = torch.zeros(100, 300, device="cuda")
    with pytest.raises(_lib.NkmxError, match="workspace"):
        mx.cu_fn_mx4_linear_e(torch.zeros(100, 4, device="cuda"), big, c, s,
                              workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(_lib.NkmxError, match="overlaps"):
        mx.cu_fn_mx4_linear_e(big[:, :4], big, c, s)
    with pytest.raises(_lib.NkmxError, match="aligned"):
        raw = torch.zeros(4 * 192 + 8, dtype=torch.uint8, device="cuda")
        mx.cu_fn_mx4_dequantize_e(x, raw[8:].view(4, 192), s)


def test_codes_behind_four_gigabytes():
    """Rows whose numbers, codes and results lie past 2^32 bytes."""
    rows, cols = 131072 + 3, 16384 + 40
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2:] = values(9, 2, cols, torch.bfloat16)
    c, s = mx.mx4_empty(rows, cols)
    mx.cu_fn_mx4_quantize_e(x, c, s)
    assert_codes(c[-2:], s[-2:], f64(x[-2:]))
    assert not c[:-2].any()
    x.fill_(1)
    mx.cu_fn_mx4_dequantize_e(x, c, s)
    want = ref.mx4_decode(c[-2:].cpu().numpy(), s[-2:].cpu().numpy(), cols)
    assert np.array_equal(f64(x[-2:]), want)
    assert not x[:-2].any()


def test_a_contracted_length_beyond_the_tiles_reach():
    """More than 2^24 columns and more rows than the smallest kernel takes: codes that are zero but for a few columns."""
    m, n, k = 40, 2064, (1 << 24) + 300
    steps = ref.steps_of(k)
    ca, sa = torch.zeros(m, steps * 64, dtype=torch.uint8, device="cuda"), torch.full((m, steps * 4), 127, dtype=torch.uint8, device="cuda")
    cb, sb = torch.zeros(n, steps * 64, dtype=torch.uint8, device="cuda"), torch.full((n, steps * 4), 127, dtype=torch.uint8, device="cuda")
    a, b = np.zeros((m, 6)), np.zeros((n, 6))
    rng = np.random.default_rng(1)
    for i, col in enumerate((0, 4097, 1 << 20, (1 << 24) - 1, 1 << 24, k - 1)):
        for codes, vals in ((ca, a), (cb, b)):
            c = rng.integers(0, 16, codes.shape[0])
            codes[:, col // 2] |= torch.from_numpy((c << (4 * (col % 2))).astype(np.uint8)).cuda()
            vals[:, i] = ref.GRID[c & 7] * np.where(c & 8, -1, 1)
    y = torch.empty(m, n, device="cuda")
    mx.cu_fn_mx4_matmul_e(y, ca, sa, cb, sb)
    assert np.array_equal(f64(y), a @ b.T)  # six products of at most 36: exact


def test_many_rows_without_columns():
    m = 3_000_000
    bias = torch.arange(3.0, device="cuda")
    y = torch.full((m, 3), 7.0, device="cuda")
    mx.cu_fn_mx4_matmul_e(y, *mx.mx4_empty(m, 0), *mx.mx4_empty(3, 0), bias=bias)
    assert torch.equal(y, bias.expand(m, 3))


@pytest.mark.parametrize("m,n,k", [(1, 16500, 4100), (16, 34000, 2000), (9, 4111, 16600)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_few_rows_against_a_large_matrix(m, n, k, dtype):
    """Two steps of k at a time, 33, 16 and 130 of them; a block of NaN stays in its row of b."""
    g = torch.Generator(device="cuda").manual_seed(m)

    def made(rows, scale):
        c, s = mx.mx4_empty(rows, k)
        mx.cu_fn_mx4_quantize_e(torch.randn(rows, k, device="cuda", generator=g) * scale, c, s)
        v = torch.empty(rows, k, device="cuda")
        mx.cu_fn_mx4_dequantize_e(v, c, s)
        return c, s, v.double()

    ca, sa, a = made(m, 1.0)
    cb, sb, b = made(n, 0.05)
    y = torch.empty(m, n, dtype=dtype, device="cuda")
    mx.cu_fn_mx4_matmul_e(y, ca, sa, cb, sb)
    bt = b.t().contiguous()
    want = a @ bt
    assert_within(y, f64(want), product_bound_of(f64(a.abs() @ bt.abs()), f64(want), k, dtype), "matmul")
    bad = [7, 15, n - 1]
    sb[bad, 5] = 255
    z = torch.empty_like(y)
    mx.cu_fn_mx4_matmul_e(z, ca, sa, cb, sb)
    assert bool(torch.isnan(z[:, bad]).all())
    z[:, bad] = y[:, bad]
    assert torch.equal(z, y)


def product_bound_of(mags, want, k, dtype):
    r = (128 + k / 64 + 8) * 2.0 ** -23 * mags
    return r + half_step(dtype) * (np.abs(want) + r) + (2.0 ** -25 if dtype == torch.float16 else 0)
