"""8-bit activation checkpoints against the numpy reference in 64 bits: save, load, the activation's gradient and the
weight gradient."""
import numpy as np
import pytest
import torch

import mx_ref as ref
from mx_gpu import DTYPES, assert_within, f64, half_step, matmul64, name, packed8, untouched, values, widened
from necklace_amd import _lib
from necklace_amd.cuda import mx

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 31), (3, 33), (7, 127), (5, 128), (4, 129), (33, 1000), (257, 64), (1, 5000), (1025, 96)]


def smallest(dtype):
    """Half the distance of the type's smallest numbers."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -127


# The normal distribution by its formula: 1.5e-7 / 2 of its own, a polynomial whose terms' magnitudes sum to 4.5 with 4
# roundings of 2^-24 each and the reciprocal's 2^-23 (together below 5.5e-7 after the factor 1/2), the exponential's
# 2^-23 and its argument's (below 1e-7): 7.5e-7 at most.
PHI = 7.5e-7


def fn_bound(x, want, fn, dtype):
    if fn == "gelu":
        own = np.abs(x) * PHI + 2.0 ** -22 * np.abs(want)
    else:  # the exponential's argument is off by |x| 2^-23, and 6 roundings of 2^-23 follow
        own = np.abs(want) * (np.abs(x) + 6) * 2.0 ** -23 + 1e-30
    return own + half_step(dtype) * (np.abs(want) + own) + smallest(dtype)


def slope_bound(x, dy, want, fn, dtype):
    if fn == "gelu":
        own = np.abs(dy) * (PHI + 2.5e-7)
    else:
        own = np.abs(dy) * (1e-30 + (np.abs(x) + 6) * 2.0 ** -23 * 2 * (1 + np.abs(x)) / (1 + np.exp(-x)))
    return own + half_step(dtype) * (np.abs(want) + own) + smallest(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("fn", [None, "gelu", "silu"])
def test_save(rows, cols, dtype, fn):
    x, _ = widened(values(rows * 3 + cols, rows, cols, dtype, 0.5), 1, 4)
    c, s = mx.act8_empty(rows, cols)
    c.fill_(99)
    s.fill_(99)
    y, wide = widened(torch.zeros(rows, cols, dtype=dtype, device="cuda"), 5, 2)
    mx.cu_fn_act8_save_e(x, c, s, Y=y if fn else None, fn=fn)
    wc, ws = ref.act8_quantize(f64(x))
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(c.cpu().numpy(), wc)
    if fn:
        want = ref.activation(f64(x), fn)
        assert_within(y, want, fn_bound(f64(x), want, fn, dtype), fn)
        assert untouched(wide, 5, cols)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_load_any_codes(rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    steps = ref.steps_of(cols)
    c = rng.integers(-128, 128, (rows, steps * 128)).astype(np.int8)
    s = rng.integers(0, 249, (rows, steps * 4), dtype=np.uint8)
    s[0, 0] = 255
    want = torch.from_numpy(ref.act8_decode(c, s, cols)).to(torch.float32).to(dtype).double().numpy()
    out, wide = widened(torch.zeros(rows, cols, dtype=dtype, device="cuda"))
    mx.cu_fn_act8_load_e(out, torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda())
    assert np.array_equal(f64(out), want, equal_nan=True)
    assert untouched(wide, 3, cols)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("fn", [None, "gelu", "silu"])
def test_save_of_extreme_blocks(dtype, fn):
    """Subnormal blocks, the type's largest numbers, ties, zeros of both signs, infinities and NaN."""
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal
    rows = [[fi.max, -fi.max, fi.max / 2], [tiny, tiny / 2, -tiny / 4], [tiny * 60, tiny * .75], [127.75, -127.75, 127.5],
            [100, .5, 1.5, 2.5, -.5, -1.5], [0.0, -0.0], [float("inf"), 1], [-float("inf"), 1], [float("nan"), 1], [-1e4, 1e4],
            [-90.0, -104.0, 88.0]]
    x = torch.zeros(len(rows), 40, dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64)
    x = x.to(dtype).cuda()
    c, s = mx.act8_empty(*x.shape)
    y = torch.empty_like(x) if fn else None
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn=fn)
    wc, ws = ref.act8_quantize(f64(x))
    assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(c.cpu().numpy(), wc)
    if fn:
        fine = torch.isfinite(x).cpu().numpy()
        with np.errstate(over="ignore", invalid="ignore"):
            want = ref.activation(f64(x), fn)
        got = f64(y)
        assert_within(got[fine], want[fine], fn_bound(f64(x)[fine], want[fine], fn, dtype), fn)
        assert got[6, 0] == np.inf and np.isnan(got[8, 0])
    out = torch.empty_like(x)
    mx.cu_fn_act8_load_e(out, c, s)
    # what the type cannot hold of the codes' values rounds to it (fp16 only)
    want = torch.from_numpy(ref.act8_decode(wc, ws, 40)).to(torch.float32).to(dtype).double().numpy()
    assert np.array_equal(f64(out), want, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("fn", ["gelu", "silu"])
def test_grad(rows, cols, dtype, fn):
    c, s, x = packed8(values(rows + cols, rows, cols, dtype, 0.5))
    dy, _ = widened(values(rows + 1, rows, cols, dtype), 2, 1)
    dx, wide = widened(torch.zeros(rows, cols, dtype=dtype, device="cuda"))
    mx.cu_fn_act8_grad_e(dx, dy, c, s, fn)
    want = f64(dy) * ref.slope(x, fn)
    assert_within(dx, want, slope_bound(x, f64(dy), want, fn, dtype), fn)
    assert untouched(wide, 3, cols)


@pytest.mark.parametrize("fn", ["gelu", "silu"])
def test_grad_against_differences(fn):
    """The derivative of what save writes, by central differences of the 64-bit function at the checkpoint's values."""
    c, s, x = packed8(values(1, 20, 100, torch.float32, 0.3))
    dy = torch.ones(20, 100, device="cuda")
    dx = torch.empty_like(dy)
    mx.cu_fn_act8_grad_e(dx, dy, c, s, fn)
    h = 1e-4  # differences are off by h^2 / 6 of the third derivative (at most 1 here) and 1e-12 / h of rounding
    want = (ref.activation(x + h, fn) - ref.activation(x - h, fn)) / (2 * h)
    assert_within(dx, want, slope_bound(x, 1.0, want, fn, torch.float32) + h * h + 1e-12 * (1 + np.abs(x)) / h)


def test_in_place_forms():
    x = values(1, 50, 300, torch.bfloat16)
    c, s = mx.act8_empty(50, 300)
    y = torch.empty_like(x)
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn="gelu")
    z, c2, s2 = x.clone(), torch.empty_like(c), torch.empty_like(s)
    mx.cu_fn_act8_save_e(z, c2, s2, Y=z, fn="gelu")
    assert torch.equal(y, z) and torch.equal(c, c2) and torch.equal(s, s2)
    mx.cu_fn_act8_grad_e(y, x, c, s, "silu")
    z = x.clone()
    mx.cu_fn_act8_grad_e(z, z, c, s, "silu")
    assert torch.equal(y, z)
    # two column ranges of one matrix
    wide = torch.zeros(50, 700, dtype=torch.bfloat16, device="cuda")
    wide[:, :300] = x
    mx.cu_fn_act8_save_e(wide[:, :300], c2, s2, Y=wide[:, 300:600], fn="silu")
    mx.cu_fn_act8_save_e(x, c, s, Y=y, fn="silu")
    assert torch.equal(wide[:, 300:600], y) and torch.equal(wide[:, :300], x) and not wide[:, 600:].any()


# ---- weight gradient.  Products are exact; an instruction sums 16 of them, one addition follows for each of a dy
# number's 1, 2 or 3 parts, 16 tokens at a time, and one per part of a split t: at most (16 + parts * t / 16 + 256 + 1) *
# 2^-23 of the sum of magnitudes.  db: at most t / 4 + 8 additions in a thread, 8 to join, the parts.

def wgrad_bounds(dy, x, t, dtype):
    mags = matmul64(np.abs(dy).T, np.abs(x))
    parts = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    return ((16 + parts * t / 16 + 257) * 2.0 ** -23 * mags,
            (t / 4 + 16 + 257) * 2.0 ** -24 * np.abs(dy).sum(0))


WGRADS = [(1, 1, 1), (1, 64, 64), (7, 3, 5), (31, 65, 33), (64, 256, 256), (65, 130, 129), (200, 63, 640), (513, 100, 100),
          (1000, 257, 300), (5001, 200, 150), (4100, 1023, 515), (11000, 1100, 1090), (20000, 40, 70)]


@pytest.mark.parametrize("t,n,k", WGRADS)
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_wgrad(t, n, k, dtype):
    c, s, x = packed8(values(t, t, k, dtype))
    dy, _ = widened(values(n, t, n, dtype, 0.01), 1, 2)
    dw, wide = widened(torch.zeros(n, k, device="cuda"))
    db = torch.full((n,), float("nan"), device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d64 = f64(dy)
    bound_w, bound_b = wgrad_bounds(d64, x, t, dtype)
    want = matmul64(d64.T, x)
    assert_within(dw, want, bound_w, "dw")
    assert_within(db, d64.sum(0), bound_b, "db")
    assert untouched(wide, 3, k)
    # again, onto what is there; and without the bias
    first, first_b = dw.clone(), db.clone()
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db, accumulate=True)
    assert_within(dw, 2 * want, 2 * bound_w + 2.0 ** -23 * np.abs(want), "accumulated dw")
    assert_within(db, 2 * d64.sum(0), 2 * bound_b + 2.0 ** -23 * np.abs(d64.sum(0)), "accumulated db")
    again = torch.empty(n, k, device="cuda")
    mx.cu_fn_act8_wgrad_e(again, dy, c, s)
    assert torch.equal(again, first)
    mx.cu_fn_act8_wgrad_e(again, dy, c, s, DB=db)
    assert torch.equal(again, first) and torch.equal(db, first_b)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_wgrad_of_numbers_over_the_type_s_range(dtype):
    """dy with small and the largest numbers next to 1: the parts it is cut into lose nothing (a part is a bf16 number:
    fp32 keeps all its bits from 2^-110 up)."""
    fi = torch.finfo(dtype)
    t, n = 32, 40
    dy = torch.zeros(t, n, dtype=dtype)
    small = fi.smallest_normal * (2.0 ** 20 if dtype == torch.float32 else 8) * (1 + fi.eps)
    vals = torch.tensor([1 + fi.eps, -(2 - fi.eps), fi.max, -fi.max, small, 1 / 3, -1e-3], dtype=torch.float64)
    for j in range(n):
        dy[j % t, j] = vals[j % len(vals)].to(dtype)  # one product each: no sum to round
    x = torch.zeros(t, 32)
    x[:, 0] = 1
    x[:, 3] = .25
    c, s, x64 = packed8(x)
    dw = torch.empty(n, 32, device="cuda")
    db = torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy.cuda(), c, s, DB=db)
    assert np.array_equal(f64(dw), f64(dy).T @ x64)
    assert np.array_equal(f64(db), f64(dy).sum(0))


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("t", [40, 3000])
def test_wgrad_with_nan_and_infinity(dtype, t):
    """A NaN or infinity reaches the results of its row and column and no other."""
    x = values(2, t, 96, dtype)
    x[:, :32] = 1  # no zero meets the infinity
    c, s, _ = packed8(x)
    dy = values(3, t, 50, dtype)
    dy[5, 7], dy[t - 1, 20] = float("nan"), float("inf")
    dw = torch.empty(50, 96, device="cuda")
    db = torch.empty(50, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    assert torch.isnan(dw[7]).all() and torch.isnan(db[7])
    assert (dw[20, :32] == float("inf")).all() and db[20] == float("inf")
    rest = [i for i in range(50) if i not in (7, 20)]
    assert torch.isfinite(dw[rest]).all() and torch.isfinite(db[rest]).all()
    # a block of the checkpoint that held a NaN
    x[4, 40] = float("nan")
    c, s, _ = packed8(x)
    dy = values(3, t, 50, dtype)
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s)
    assert torch.isnan(dw[:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_wgrad_against_differences(dtype):
    """The loss sum(dy * (x^ W^T + b)) is linear in W and b: its differences are its gradient."""
    c, s, x = packed8(values(1, 60, 40, dtype))
    dy = values(2, 60, 30, dtype)
    dw, db = torch.empty(30, 40, device="cuda"), torch.empty(30, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d64 = f64(dy)
    bound_w, bound_b = wgrad_bounds(d64, x, 60, dtype)
    loss = lambda w, b: float((d64 * (x @ w.T + b)).sum())  # noqa: E731
    w, b = np.zeros((30, 40)), np.zeros(30)
    scale = np.abs(d64).sum() * max(1.0, np.abs(x).max())
    for i, j in ((0, 0), (3, 17), (29, 39)):
        step = np.zeros_like(w)
        step[i, j] = 1
        assert abs(loss(w + step, b) - loss(w - step, b) - 2 * float(dw[i, j])) <= 2 * bound_w[i, j] + 1e-13 * scale
    step = np.zeros_like(b)
    step[4] = 1
    assert abs(loss(w, b + step) - loss(w, b - step) - 2 * float(db[4])) <= 2 * bound_b[4] + 1e-13 * scale


def test_wgrad_of_no_tokens_and_no_columns():
    dw, db = torch.full((5, 40), 3.0, device="cuda"), torch.full((5,), 2.0, device="cuda")
    c, s = mx.act8_empty(0, 40)
    dy = torch.empty(0, 5, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db, accumulate=True)
    assert (dw == 3).all() and (db == 2).all()
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    assert not dw.any() and not db.any()
    dy = torch.ones(3000, 5, device="cuda")
    c, s = mx.act8_empty(3000, 0)
    mx.cu_fn_act8_wgrad_e(torch.empty(5, 0, device="cuda"), dy, c, s, DB=db)
    assert (db == 3000).all()


def test_refusals_of_tensors_that_do_not_fit():
    x = torch.zeros(4, 300, device="cuda")
    c, s = mx.act8_empty(4, 300)
    with pytest.raises(ValueError, match="does not match"):
        mx.cu_fn_act8_save_e(x[:3], c, s)
    with pytest.raises(TypeError, match="int8"):
        mx.cu_fn_act8_save_e(x, c.view(torch.uint8), s)
    with pytest.raises(ValueError, match="activation"):
        mx.cu_fn_act8_save_e(x, c, s, Y=x)
    with pytest.raises(TypeError, match="Y: expected"):
        mx.cu_fn_act8_save_e(x, c, s, fn="gelu")
    with pytest.raises(TypeError, match="Y is"):
        mx.cu_fn_act8_save_e(x, c, s, Y=x.bfloat16(), fn="gelu")
    with pytest.raises(ValueError, match="Y is"):
        mx.cu_fn_act8_save_e(x, c, s, Y=x[:, 1:], fn="gelu")
    with pytest.raises(ValueError, match="DY is"):
        mx.cu_fn_act8_grad_e(x, x[:, 1:], c, s, "gelu")
    with pytest.raises(_lib.NkmxError, match="overlaps"):
        flat = torch.zeros(1300, device="cuda")
        mx.cu_fn_act8_grad_e(flat[:1200].view(4, 300), flat[4:1204].view(4, 300), c, s, "gelu")
    dw = torch.zeros(7, 300, device="cuda")
    dy = torch.zeros(4, 7, device="cuda")
    with pytest.raises(TypeError, match="DW"):
        mx.cu_fn_act8_wgrad_e(dw.bfloat16(), dy, c, s)
    with pytest.raises(ValueError, match="DY has"):
        mx.cu_fn_act8_wgrad_e(dw, dy[:, :6], c, s)
    with pytest.raises(ValueError, match="does not match"):
        mx.cu_fn_act8_wgrad_e(dw, dy[:3], c, s)
    with pytest.raises(ValueError, match="DB"):
        mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=torch.zeros(6, device="cuda"))
    with pytest.raises(TypeError, match="DB"):
        mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=torch.zeros(7, device="cuda", dtype=torch.float16))
    with pytest.raises(_lib.NkmxError, match="overlaps"):
        mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=dw.view(-1)[:7])


def test_checkpoints_behind_four_gigabytes():
    rows, cols = 131072 + 3, 32768 + 40
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2:] = values(9, 2, cols, torch.bfloat16)
    c, s = mx.act8_empty(rows, cols)
    mx.cu_fn_act8_save_e(x, c, s)
    wc, ws = ref.act8_quantize(f64(x[-2:]))
    assert np.array_equal(c[-2:].cpu().numpy(), wc) and np.array_equal(s[-2:].cpu().numpy(), ws)
    dy = torch.ones(rows, 3, dtype=torch.bfloat16, device="cuda")
    dw = torch.empty(3, cols, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s)
    x64 = ref.act8_decode(wc, ws, cols)
    assert_within(dw, np.tile(x64.sum(0), (3, 1)), 2.0 ** -22 * np.abs(x64).sum(0))
    mx.cu_fn_act8_load_e(x, c, s)
    assert np.array_equal(f64(x[-2:]), x64) and not x[:-2].any()


@pytest.mark.parametrize("dtype,ld", [(torch.bfloat16, 1 << 24), (torch.float32, 1 << 26)], ids=["bfloat16", "float32"])
def test_wgrad_of_gradients_whose_rows_lie_far_apart(dtype, ld):
    """Rows of dy whose distances within a tile pass 2^31 and 2^32 bytes."""
    t, n, k = 150, 70, 40
    wide = torch.empty(t, ld, dtype=dtype, device="cuda")
    dy = wide[:, 1000:1000 + n]
    dy.copy_(values(4, t, n, dtype))
    c, s, x = packed8(values(5, t, k, dtype))
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d64 = f64(dy)
    bound_w, bound_b = wgrad_bounds(d64, x, t, dtype)
    assert_within(dw, matmul64(d64.T, x), bound_w, "dw")
    assert_within(db, d64.sum(0), bound_b, "db")


@pytest.mark.parametrize("left", [0, 1, 2, 3])
@pytest.mark.parametrize("t,n,k", [(200, 130, 140), (3000, 300, 130), (9000, 520, 520)])
def test_wgrad_of_bf16_gradients_at_any_start(t, n, k, left):
    """Even starts and leading dimensions take dy to LDS as it lies in memory, odd ones through registers."""
    for more in (0, 1):
        wide = torch.full((t, n + left + 2 + more), float("nan"), dtype=torch.bfloat16, device="cuda")
        dy = wide[:, left:left + n]
        dy.copy_(values(t, t, n, torch.bfloat16, 0.1))
        c, s, x = packed8(values(7, t, k, torch.bfloat16))
        dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
        mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
        d64 = f64(dy)
        bound_w, bound_b = wgrad_bounds(d64, x, t, torch.bfloat16)
        assert_within(dw, matmul64(d64.T, x), bound_w, "dw")
        assert_within(db, d64.sum(0), bound_b, "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_wgrad_of_a_few_tiles_more_than_cus(dtype):
    """258 tiles of 256: t is cut so that the rounds come out evenly."""
    t, n, k = 3000, 257, 32900
    assert mx.act8_wgrad_workspace(dtype, t, n, k) >= 2 * 4 * n * k
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(t, k, device="cuda", generator=g)
    c, s = mx.act8_empty(t, k)
    mx.cu_fn_act8_save_e(x, c, s)
    mx.cu_fn_act8_load_e(x, c, s)
    dy = torch.randn(t, n, device="cuda", generator=g).to(dtype)
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d64, x64 = dy.double().t().contiguous(), x.double()
    parts = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    bound = (16 + parts * t / 16 + 257) * 2.0 ** -23 * (d64.abs() @ x64.abs())
    assert bool(((dw.double() - d64 @ x64).abs() <= bound).all())
    assert bool(((db.double() - d64.sum(1)).abs() <= (t / 4 + 16 + 257) * 2.0 ** -24 * d64.abs().sum(1)).all())


@pytest.mark.parametrize("t,n,k", [(300, 1800, 2000), (2100, 64, 64), (700, 640, 650), (260, 70, 4100), (16384, 66, 130)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_wgrad_of_contiguous_gradients(t, n, k, dtype):
    """Tiles of 128 without a cut, of 64 with few and with many stages a part; the same bits again and without the bias."""
    g = torch.Generator(device="cuda").manual_seed(t)
    x = torch.randn(t, k, device="cuda", generator=g)
    c, s = mx.act8_empty(t, k)
    mx.cu_fn_act8_save_e(x, c, s)
    mx.cu_fn_act8_load_e(x, c, s)
    dy = torch.randn(t, n, device="cuda", generator=g).to(dtype)
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db)
    d64 = f64(dy)
    bound_w, bound_b = wgrad_bounds(d64, f64(x), t, dtype)
    assert_within(dw, matmul64(d64.T, f64(x)), bound_w, "dw")
    assert_within(db, d64.sum(0), bound_b, "db")
    again = torch.empty_like(dw)
    mx.cu_fn_act8_wgrad_e(again, dy, c, s)
    assert torch.equal(again, dw)
