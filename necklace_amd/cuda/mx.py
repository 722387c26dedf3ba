"""Microscaled storage on MI355X: 4-bit floating point with its products, 8-bit activation checkpoints.

Beside the 2-bit gradient quantizer (quantize.py) and in its manner: the caller brings every tensor, the work
is done by the HIP kernels of libnkmx.so (include/nkmx.h has the formats bit by bit), calls run on torch's
current stream or on `stream` and block unless ``sync=False``.

A matrix [rows, cols] is packed along its rows: blocks of 32 neighbouring columns share a power of two as their
scale, rows are padded with zeros to whole steps of 128 columns.

* mx4: codes uint8 [rows, steps * 64] (2 a byte, the even column in the low half), values 0, .5, 1, 1.5, 2, 3, 4, 6
  times the scale with a sign; `mx4_empty` makes the tensors;
* act8: codes int8 [rows, steps * 128], whole numbers -127 .. 127 times the scale; `act8_empty`;
* both: scales uint8 [rows, steps * 4], exponent + 127; 255 marks a block that held an infinity or a NaN: it decodes
  to NaN.  A value is off by at most half the distance of the codes around it: for act8 2^e / 2 (2^e where the
  largest magnitude of a block would round to 128), for mx4 2^e / 4 below 2 scales, 2^e / 2 from there to 4, 2^e from
  there to 6; beyond, where 6 is the last code, less than 2 * 2^e.

Tensors of numbers are float32, bfloat16 or float16 and may be column ranges of wider matrices (any leading
dimension, columns next to each other); more than two dimensions are taken as rows of the last one where that needs
no copy, one dimension as a single row.  Outputs may not overlap inputs unless a call says so.
"""
import functools

import torch

from .. import _lib
from . import nbutils
from .quantize import _finish

BLOCK = 32
STEP = 128

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FNS = {None: 0, "gelu": 1, "silu": 2}


def steps_of(cols):
    """Steps of 128 columns of a packed row."""
    return (cols + STEP - 1) // STEP


def mx4_empty(rows, cols, device="cuda"):
    """Codes and scales for the mx4 of a [rows, cols] matrix."""
    s = steps_of(cols)
    return (torch.empty(rows, s * 64, dtype=torch.uint8, device=device),
            torch.empty(rows, s * 4, dtype=torch.uint8, device=device))


def act8_empty(rows, cols, device="cuda"):
    """Codes and scales for the act8 of a [rows, cols] matrix."""
    s = steps_of(cols)
    return (torch.empty(rows, s * STEP, dtype=torch.int8, device=device),
            torch.empty(rows, s * 4, dtype=torch.uint8, device=device))


def shape2(t):
    """(rows, cols) of a tensor taken as rows of its last dimension."""
    if t.dim() == 2:
        return t.shape[0], t.shape[1]
    if t.dim() == 0:
        raise TypeError("expected at least 1 dimension")
    rows = 1
    for n in t.shape[:-1]:
        rows *= n
    return rows, t.shape[-1]


def row_stride(t):
    """Distance of neighbouring rows in elements, None where the tensor is not rows of neighbouring columns."""
    rows, cols = shape2(t)
    if rows == 0 or cols == 0:
        return cols
    if cols > 1 and t.stride(-1) != 1:
        return None
    ld = None
    want = None
    for d in range(t.dim() - 2, -1, -1):  # the dimensions above the last one, innermost first
        if t.shape[d] == 1:
            continue
        if ld is None:
            ld = t.stride(d)
        elif t.stride(d) != want:
            return None
        want = t.stride(d) * t.shape[d]
    if ld is None:
        return cols
    return ld if ld >= cols else None


def _matrix(name, t):
    """(rows, columns, leading dimension) of a tensor of numbers."""
    try:
        if t.dim() == 2 and t.is_cuda and t.dtype in _TYPES:  # what nearly every call brings
            rows, cols = t.shape
            ld, one = t.stride()
            if one == 1:
                if rows == 1:
                    return 1, cols, cols
                if ld >= cols and rows > 1:
                    return rows, cols, ld
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise TypeError(f"{name}: expected a GPU tensor")
    if t.dim() == 0:
        raise TypeError(f"{name}: expected at least 1 dimension")
    ld = row_stride(t)
    if ld is None:
        raise ValueError(f"{name}: strides {tuple(t.stride())} are not rows of neighbouring columns")
    rows, cols = shape2(t)
    return rows, cols, ld


def _same_type(name, t, other, want):
    if t.dtype != want:
        raise TypeError(f"{name} is {t.dtype}, {other} is {want}")


def _packed(name, c, s, rows, cols, mx4, what):
    """Checks codes `c` and scales `s` against the matrix they stand for."""
    steps = (cols + STEP - 1) // STEP
    width, dtype = (steps * 64, torch.uint8) if mx4 else (steps * STEP, torch.int8)
    try:
        if c.shape == (rows, width) and s.shape == (rows, steps * 4) and c.dtype is dtype and s.dtype is torch.uint8 \
                and c.is_cuda and s.is_cuda and c.is_contiguous() and s.is_contiguous():
            return
    except AttributeError:
        pass
    for part, t, dtype, width in ((name, c, dtype, width), (f"scales of {name}", s, torch.uint8, steps * 4)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{part}: expected a torch tensor, got {type(t).__name__}")
        if t.dtype != dtype:
            raise TypeError(f"{part}: expected {dtype}, got {t.dtype}")
        if not t.is_cuda:
            raise TypeError(f"{part}: expected a GPU tensor")
        if tuple(t.shape) != (rows, width):
            raise ValueError(f"{part}: shape {tuple(t.shape)} does not match {(rows, width)} of {what}")
        if not t.is_contiguous():
            raise ValueError(f"{part}: must be contiguous")


def _device(first, *others):
    """Index of the GPU that all tensors are on."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError("all tensors must be on the same GPU")
    return dev


@functools.lru_cache(maxsize=4096)
def _linear_bytes(m, n, k):
    return int(_lib.mx_lib().nkmx_mx4_linear_workspace(m, n, k))


@functools.lru_cache(maxsize=4096)
def _wgrad_bytes(ty, t, n, k):
    return int(_lib.mx_lib().nkmx_act8_wgrad_workspace(ty, t, n, k))


def _workspace(given, need, dev, stream, handle):
    """`given`, or fresh memory of the stream that the call runs on."""
    if given is not None:
        if not isinstance(given, torch.Tensor) or given.dtype != torch.uint8 or not given.is_contiguous() \
                or given.get_device() != dev:
            raise TypeError("workspace: expected a contiguous uint8 tensor on the same GPU")
        return given
    if not need:
        return None
    if stream is None:
        return torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(handle, device=torch.device("cuda", dev)) if handle else torch.cuda.default_stream(dev)
    with torch.cuda.stream(stream):  # the allocator hands a block on within its own stream only
        return torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))


def _bias(bias, n, y):
    if bias is None:
        return None
    if not isinstance(bias, torch.Tensor):
        raise TypeError(f"bias: expected a torch tensor, got {type(bias).__name__}")
    _same_type("bias", bias, "Y", y.dtype)
    if bias.shape != (n,) or (n > 1 and bias.stride(0) != 1):
        raise ValueError(f"bias: expected {n} contiguous elements")
    return bias.data_ptr()


# ------------------------------------------------------------------ 4-bit floating point

def cu_fn_mx4_quantize_e(A, C, S, transpose=False, stream=None, sync=True):
    """Codes C and scales S of the matrix A, or with `transpose` of A's transpose (blocks along A's columns: the
    form that the gradient of a product's input contracts over), laid out by `mx4_empty(rows, cols)` of what is packed."""
    rows, cols, ld = _matrix("A", A)
    pr, pc = (cols, rows) if transpose else (rows, cols)
    _packed("C", C, S, pr, pc, True, "A's transpose" if transpose else "A")
    dev = _device(A, C, S)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_mx4_quantize(A.data_ptr(), _TYPES[A.dtype], rows, cols, ld, C.data_ptr(), S.data_ptr(),
                                               1 if transpose else 0, h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def cu_fn_mx4_dequantize_e(A, C, S, stream=None, sync=True):
    """Decode C, S into A (overwrite); exact in float32 and bfloat16, rounded once in float16."""
    rows, cols, ld = _matrix("A", A)
    _packed("C", C, S, rows, cols, True, "A")
    dev = _device(A, C, S)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_mx4_dequantize(A.data_ptr(), _TYPES[A.dtype], rows, cols, ld, C.data_ptr(), S.data_ptr(), h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def cu_fn_mx4_matmul_e(Y, CA, SA, CB, SB, bias=None, stream=None, sync=True):
    """Y[i, j] = sum over c of A[i, c] B[j, c] (+ bias[j]), A and B given by their codes; summed in fp32, rounded once.
    The contracted length is the packed one (the padding is zeros)."""
    m, n, ld = _matrix("Y", Y)
    if not isinstance(CA, torch.Tensor) or CA.dim() != 2 or CA.shape[1] % 64:
        raise TypeError("CA: expected codes [rows, steps * 64]")
    k = CA.shape[1] * 2
    _packed("CA", CA, SA, m, k, True, "Y and its own length")
    _packed("CB", CB, SB, n, k, True, "Y and CA")
    b = _bias(bias, n, Y)
    dev = _device(Y, CA, SA, CB, SB, bias)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_mx4_matmul(Y.data_ptr(), _TYPES[Y.dtype], m, n, k, ld, CA.data_ptr(), SA.data_ptr(),
                                             CB.data_ptr(), SB.data_ptr(), b, h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def mx4_linear_workspace(m, n, k):
    """Bytes of workspace that `cu_fn_mx4_linear_e` needs."""
    return _linear_bytes(m, n, k)


def cu_fn_mx4_linear_e(Y, X, CB, SB, bias=None, workspace=None, stream=None, sync=True):
    """Y = mx4(X) B^T (+ bias): X [m, k] is quantized on its way into the product with the packed B [n, k]; the same
    bits as `cu_fn_mx4_quantize_e` and `cu_fn_mx4_matmul_e`, in one launch for few rows.

    `workspace` (uint8, `mx4_linear_workspace` bytes; two calls that run at the same time need one each) is allocated
    by torch if it is not given."""
    m, n, ldy = _matrix("Y", Y)
    mx, k, ldx = _matrix("X", X)
    _same_type("X", X, "Y", Y.dtype)
    if mx != m:
        raise ValueError(f"X has {mx} rows, Y {m}")
    _packed("CB", CB, SB, n, k, True, "Y's columns and X's")
    b = _bias(bias, n, Y)
    dev = _device(Y, X, CB, SB, bias)
    L = _lib.mx_lib()
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        ws = _workspace(workspace, _linear_bytes(m, n, k), dev, stream, h)
        code = L.nkmx_mx4_linear(Y.data_ptr(), X.data_ptr(), _TYPES[Y.dtype], m, n, k, ldy, ldx, CB.data_ptr(),
                                 SB.data_ptr(), b, ws.data_ptr() if ws is not None else None,
                                 ws.numel() if ws is not None else 0, h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


# ------------------------------------------------------------------ 8-bit activation checkpoints

def _fn_code(fn, none_allowed):
    if fn not in _FNS or (fn is None and not none_allowed):
        raise ValueError(f"fn: expected {'None, ' if none_allowed else ''}'gelu' or 'silu', got {fn!r}")
    return _FNS[fn]


def cu_fn_act8_save_e(A, C, S, Y=None, fn=None, stream=None, sync=True):
    """Checkpoint A in 8 bits (C, S from `act8_empty`) and, with `fn` ("gelu": x Phi(x), "silu": x / (1 + e^-x)), write
    Y = fn(A) in the same pass, taken of A itself.  Y may be A.  With an activation, C and S may both be None: Y alone is
    written, the same bits."""
    f = _fn_code(fn, True)
    rows, cols, ld = _matrix("A", A)
    saves = fn is None or C is not None or S is not None
    if saves:
        _packed("C", C, S, rows, cols, False, "A")
    y, ldy = None, 0
    if fn is not None:
        yr, yc, ldy = _matrix("Y", Y)
        _same_type("Y", Y, "A", A.dtype)
        if (yr, yc) != (rows, cols):
            raise ValueError(f"Y is {yr} x {yc}, A {rows} x {cols}")
        y = Y.data_ptr()
    elif Y is not None:
        raise ValueError("Y is written with an activation `fn` only")
    dev = _device(A, C, S, Y)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_act8_save(A.data_ptr(), y, _TYPES[A.dtype], f, rows, cols, ld, ldy,
                                            C.data_ptr() if saves else None, S.data_ptr() if saves else None, h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def cu_fn_act8_load_e(A, C, S, stream=None, sync=True):
    """Decode the checkpoint C, S into A (overwrite); exact in float32 and bfloat16, rounded once in float16."""
    rows, cols, ld = _matrix("A", A)
    _packed("C", C, S, rows, cols, False, "A")
    dev = _device(A, C, S)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_act8_load(A.data_ptr(), _TYPES[A.dtype], rows, cols, ld, C.data_ptr(), S.data_ptr(), h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def cu_fn_act8_grad_e(DX, DY, C, S, fn, stream=None, sync=True):
    """DX = DY * fn'(x), x read from its checkpoint C, S.  DX may be DY."""
    f = _fn_code(fn, False)
    rows, cols, lddx = _matrix("DX", DX)
    dr, dc, lddy = _matrix("DY", DY)
    _same_type("DY", DY, "DX", DX.dtype)
    if (dr, dc) != (rows, cols):
        raise ValueError(f"DY is {dr} x {dc}, DX {rows} x {cols}")
    _packed("C", C, S, rows, cols, False, "DX")
    dev = _device(DX, DY, C, S)
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        code = _lib.mx_lib().nkmx_act8_grad(DX.data_ptr(), DY.data_ptr(), _TYPES[DX.dtype], f, rows, cols, lddx, lddy,
                                            C.data_ptr(), S.data_ptr(), h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)


def act8_wgrad_workspace(dtype, t, n, k):
    """Bytes of workspace that `cu_fn_act8_wgrad_e` needs for gradients DY of `dtype`."""
    return _wgrad_bytes(_TYPES[dtype], t, n, k)


def cu_fn_act8_wgrad_e(DW, DY, C, S, DB=None, accumulate=False, workspace=None, stream=None, sync=True):
    """Weight gradient of a linear layer from the checkpoint of its input: DW[j, c] = sum over i of DY[i, j] x[i, c],
    x [t, k] given by C, S.  DW is float32 [n, k], DY [t, n] of any of the types; DB (float32 [n]) gets the sums of DY's
    columns (alone, where k is 0).  ``accumulate=True`` adds to what DW and DB hold.  Products are exact and sums fp32 for
    every type; the result is the same bits every time.  `workspace` as in `cu_fn_mx4_linear_e`, of `act8_wgrad_workspace`
    bytes."""
    n, k, lddw = _matrix("DW", DW)
    if DW.dtype != torch.float32:
        raise TypeError(f"DW: expected float32, got {DW.dtype}")
    t, dn, lddy = _matrix("DY", DY)
    if dn != n:
        raise ValueError(f"DY has {dn} columns, DW {n} rows")
    _packed("C", C, S, t, k, False, "DY's rows and DW's columns")
    db = None
    if DB is not None:
        if not isinstance(DB, torch.Tensor) or DB.dtype != torch.float32:
            raise TypeError("DB: expected a float32 tensor")
        if DB.shape != (n,) or (n > 1 and DB.stride(0) != 1):
            raise ValueError(f"DB: expected {n} contiguous elements")
        db = DB.data_ptr()
    dev = _device(DW, DY, C, S, DB)
    L = _lib.mx_lib()
    ty = _TYPES[DY.dtype]
    with nbutils.on_device(dev):
        h = nbutils.stream_handle(stream, dev)
        ws = _workspace(workspace, _wgrad_bytes(ty, t, n, k), dev, stream, h)
        code = L.nkmx_act8_wgrad(DW.data_ptr(), db, DY.data_ptr(), ty, t, n, k, lddw, lddy, C.data_ptr(), S.data_ptr(),
                                 1 if accumulate else 0, ws.data_ptr() if ws is not None else None,
                                 ws.numel() if ws is not None else 0, h)
        if code:
            _lib.check_mx(code)
        _finish(stream, dev, sync)
