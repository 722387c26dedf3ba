"""libnkmx.so exports what include/nkmx.h declares and refuses bad arguments before touching a GPU; the Python layer's
own refusals.  No kernel is launched here."""
import ctypes as ct
import os
import re

import pytest
import torch

from conftest import ROOT
from necklace_amd import _lib
from necklace_amd.cuda import mx

P = 1 << 20  # an address that is never read


def _declared():
    text = open(os.path.join(ROOT, "include", "nkmx.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(nkmx_[a-z0-9_]+)\s*\(", text)))


def test_every_declared_symbol_is_exported_and_bound():
    L = _lib.mx_lib()
    assert sorted(_lib.MX_SYMBOLS) == _declared()
    for n in _declared():
        assert hasattr(L, n)
    text = open(os.path.join(ROOT, "include", "nkmx.h")).read()
    assert L.nkmx_version() == int(re.search(r"#define NKMX_VERSION (\d+)", text).group(1))


def test_every_error_has_a_text():
    L = _lib.mx_lib()
    texts = {L.nkmx_strerror(c) for c in range(0, -6, -1)}
    assert len(texts) == 6 and b"nkmx: unknown error" not in texts
    assert L.nkmx_strerror(-99) == b"nkmx: unknown error"


FAR = 1 << 40


def _quantize(x=FAR, ty=0, rows=4, cols=300, ld=300, c=2 * FAR, s=3 * FAR, tr=0):
    return _lib.mx_lib().nkmx_mx4_quantize(x, ty, rows, cols, ld, c, s, tr, None)


def test_quantize_refusals():
    assert _quantize(rows=0) == 0 and _quantize(cols=0, ld=0) == 0 and _quantize(x=None, rows=0) == 0
    assert _quantize(x=None) == -1 and _quantize(c=None) == -1 and _quantize(s=None) == -1
    assert _quantize(x=FAR + 2) == -2 and _quantize(c=2 * FAR + 8) == -2 and _quantize(s=3 * FAR + 2) == -2
    assert _quantize(ty=3) == -3 and _quantize(ty=-1) == -3
    assert _quantize(rows=1 << 31) == -3 and _quantize(cols=1 << 31, ld=1 << 31) == -3
    assert _quantize(ld=299) == -3
    # 4 rows of 300 floats end at FAR + 4800; their codes take 4 * 192 bytes, their scales 4 * 12
    assert _quantize(c=FAR + 4784) == -4 and _quantize(c=FAR - 752) == -4
    assert _quantize(s=FAR + 4796) == -4 and _quantize(c=2 * FAR, s=2 * FAR + 764) == -4
    # the transpose: 300 rows of 1 step: 300 * 64 and 300 * 4 bytes
    assert _quantize(tr=1, c=FAR - 19184) == -4 and _quantize(tr=1, s=FAR - 1196) == -4


def test_dequantize_refusals():
    f = _lib.mx_lib().nkmx_mx4_dequantize
    assert f(FAR, 0, 0, 5, 5, None, None, None) == 0
    assert f(FAR, 1, 4, 300, 300, None, 2 * FAR, None) == -1 and f(None, 1, 4, 300, 300, FAR, 2 * FAR, None) == -1
    assert f(FAR + 1, 1, 4, 300, 300, 2 * FAR, 3 * FAR, None) == -2
    assert f(FAR, 7, 4, 300, 300, 2 * FAR, 3 * FAR, None) == -3
    assert f(FAR, 0, 4, 300, 300, FAR + 4784, 3 * FAR, None) == -4


def _matmul(y=FAR, ty=1, m=5, n=7, k=300, ld=7, ca=2 * FAR, sa=3 * FAR, cb=4 * FAR, sb=5 * FAR, bias=None):
    return _lib.mx_lib().nkmx_mx4_matmul(y, ty, m, n, k, ld, ca, sa, cb, sb, bias, None)


def test_matmul_refusals():
    assert _matmul(m=0) == 0 and _matmul(n=0) == 0
    assert _matmul(y=None) == -1 and _matmul(ca=None) == -1 and _matmul(sb=None) == -1
    assert _matmul(y=FAR + 1) == -2 and _matmul(cb=4 * FAR + 4) == -2 and _matmul(bias=6 * FAR + 1) == -2
    assert _matmul(ty=9) == -3 and _matmul(ld=6) == -3 and _matmul(k=1 << 31) == -3
    # y: 5 rows of 7 bf16 = 70 bytes
    assert _matmul(ca=FAR + 64) == -4 and _matmul(sb=FAR - 80) == -4 and _matmul(bias=FAR + 68) == -4
    # a and b may be the same matrix, and are only read: refused for another reason, after the overlap check
    assert _matmul(ca=4 * FAR, y=4 * FAR) == -4


def test_linear_refusals():
    L = _lib.mx_lib()

    def f(y=FAR, x=2 * FAR, ty=0, m=100, n=7, k=300, ldy=7, ldx=300, cb=3 * FAR, sb=4 * FAR, bias=None, ws=5 * FAR, nb=None):
        nb = L.nkmx_mx4_linear_workspace(m, n, k) if nb is None else nb
        return L.nkmx_mx4_linear(y, x, ty, m, n, k, ldy, ldx, cb, sb, bias, ws, nb, None)

    assert L.nkmx_mx4_linear_workspace(1, 4096, 4096) == 0
    need = L.nkmx_mx4_linear_workspace(100, 7, 300)
    assert need == 100 * 3 * 68
    assert f(m=0) == 0
    assert f(x=None) == -1 and f(cb=None) == -1
    assert f(ws=None) == -5 and f(nb=need - 1) == -5 and f(ws=5 * FAR + 8) == -5
    assert f(ldx=299) == -3
    assert f(y=2 * FAR) == -4 and f(ws=2 * FAR + 16) == -4 and f(ws=FAR) == -4 and f(ws=4 * FAR) == -4
    assert f(bias=5 * FAR + 100) == -4


def test_act8_refusals():
    L = _lib.mx_lib()

    def save(x=FAR, y=2 * FAR, ty=0, fn=1, rows=4, cols=300, ldx=300, ldy=300, c=3 * FAR, s=4 * FAR):
        return L.nkmx_act8_save(x, y, ty, fn, rows, cols, ldx, ldy, c, s, None)

    assert save(rows=0) == 0
    assert save(x=None) == -1 and save(y=None) == -1 and save(c=None) == -1
    assert save(y=2 * FAR + 2) == -2 and save(c=3 * FAR + 4) == -2
    assert save(fn=3) == -3 and save(fn=-1) == -3 and save(ty=4) == -3 and save(ldy=200) == -3
    assert save(y=FAR + 4) == -4            # shifted by one element: not in place
    assert save(y=FAR, ldx=300, ldy=301) == -4
    assert save(c=2 * FAR + 16) == -4 and save(s=3 * FAR) == -4
    # column ranges of one wider matrix interleave but do not overlap... unless they do
    assert save(x=FAR, y=FAR + 4 * 299, ldx=600, ldy=600) == -4

    def grad(dx=FAR, dy=2 * FAR, ty=0, fn=1, rows=4, cols=300, lddx=300, lddy=300, c=3 * FAR, s=4 * FAR):
        return L.nkmx_act8_grad(dx, dy, ty, fn, rows, cols, lddx, lddy, c, s, None)

    assert grad(rows=0) == 0
    assert grad(fn=0) == -3 and grad(dy=None) == -1 and grad(dy=FAR + 4) == -4 and grad(dx=3 * FAR) == -4
    assert L.nkmx_act8_load(3 * FAR, 0, 4, 300, 300, 3 * FAR, 4 * FAR, None) == -4
    assert L.nkmx_act8_load(None, 0, 4, 300, 300, 3 * FAR, 4 * FAR, None) == -1


def test_wgrad_refusals():
    L = _lib.mx_lib()

    def f(dw=FAR, db=None, dy=2 * FAR, ty=0, t=64, n=7, k=300, lddw=300, lddy=7, c=3 * FAR, s=4 * FAR, ws=None, nb=0):
        return L.nkmx_act8_wgrad(dw, db, dy, ty, t, n, k, lddw, lddy, c, s, 0, ws, nb, None)

    assert f(n=0) == 0 and f(k=0) == 0
    assert f(dw=None) == -1 and f(dy=None) == -1 and f(s=None) == -1
    assert f(dw=FAR + 2) == -2 and f(db=5 * FAR + 2) == -2
    assert f(ty=5) == -3 and f(lddy=6) == -3 and f(lddw=10) == -3 and f(t=1 << 31) == -3
    assert f(dw=2 * FAR) == -4 and f(db=FAR + 40) == -4 and f(db=2 * FAR + 4) == -4 and f(dw=3 * FAR + 64) == -4
    need = L.nkmx_act8_wgrad_workspace(0, 16384, 64, 64)
    assert need > 0
    big = dict(t=16384, n=64, k=64, lddw=64, lddy=64)
    assert f(**big) == -5 and f(ws=5 * FAR, nb=need - 1, **big) == -5 and f(ws=5 * FAR + 4, nb=need, **big) == -5
    assert f(ws=2 * FAR, nb=need, **big) == -4


@pytest.mark.parametrize("t,n,k", [(0, 5, 5), (1, 1, 1), (64, 256, 256), (5001, 1023, 4097), (16384, 4096, 1024),
                                   (2 ** 31 - 1, 64, 64), (100000, 8192, 8192)])
def test_wgrad_workspace_is_bounded(t, n, k):
    for ty in range(3):
        got = _lib.mx_lib().nkmx_act8_wgrad_workspace(ty, t, n, k)
        assert got % 16 == 0 and got <= 256 * (n * (k + 3) + n + 3) * 4


# ---- the Python layer

def test_sizes_of_packed_tensors():
    assert [mx.steps_of(c) for c in (0, 1, 128, 129, 1000)] == [0, 1, 1, 2, 8]
    c, s = mx.mx4_empty(3, 129, device="cpu")
    assert c.shape == (3, 128) and s.shape == (3, 8) and c.dtype == s.dtype == torch.uint8
    c, s = mx.act8_empty(3, 129, device="cpu")
    assert c.shape == (3, 256) and s.shape == (3, 8) and c.dtype == torch.int8


def test_strides_that_are_rows_of_neighbouring_columns():
    x = torch.zeros(6, 10)
    assert mx.row_stride(x) == 10 and mx.row_stride(x[:, 2:7]) == 10 and mx.row_stride(x[::2]) == 20
    assert mx.row_stride(x.t()) is None and mx.row_stride(x[:, ::2]) is None
    assert mx.row_stride(x.expand(4, 6, 10)) is None and mx.row_stride(x[:1].expand(6, 10)) is None
    assert mx.row_stride(x[0]) == 10 and mx.row_stride(x[:, :1]) == 10 and mx.row_stride(x.t()[:1]) is None
    y = torch.zeros(2, 3, 4, 5)
    assert mx.row_stride(y) == 5 and mx.row_stride(y[..., 1:4]) == 5
    assert mx.row_stride(y[:, 1:]) is None and mx.row_stride(y[:, :, 0]) == 20 and mx.row_stride(y[:, 1]) is None
    assert mx.row_stride(y[:1, 1:]) == 5
    assert mx.shape2(y) == (24, 5) and mx.shape2(x[0]) == (1, 10)
    assert mx.row_stride(torch.zeros(0, 7)) == 7 and mx.shape2(torch.zeros(2, 0, 7)) == (0, 7)


def test_host_tensors_and_wrong_types_are_refused():
    c, s = mx.mx4_empty(4, 8, device="cpu")
    x = torch.zeros(4, 8)
    for call in (lambda: mx.cu_fn_mx4_quantize_e(x, c, s), lambda: mx.cu_fn_mx4_dequantize_e(x, c, s),
                 lambda: mx.cu_fn_mx4_matmul_e(x, c, s, c, s), lambda: mx.cu_fn_mx4_linear_e(x, x, c, s),
                 lambda: mx.cu_fn_act8_save_e(x, c, s), lambda: mx.cu_fn_act8_load_e(x, c, s),
                 lambda: mx.cu_fn_act8_grad_e(x, x, c, s, "gelu"), lambda: mx.cu_fn_act8_wgrad_e(x, x, c, s)):
        with pytest.raises(TypeError, match="GPU tensor"):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        mx.cu_fn_mx4_quantize_e([1.0], c, s)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        mx.cu_fn_mx4_quantize_e(x.double(), c, s)
    for fn in ("relu", "", 1):
        with pytest.raises(ValueError, match="fn"):
            mx.cu_fn_act8_save_e(x, c, s, Y=x, fn=fn)
    with pytest.raises(ValueError, match="fn"):
        mx.cu_fn_act8_grad_e(x, x, c, s, None)
