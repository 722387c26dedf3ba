"""The microscaled formats and operators in numpy, 64 bits, straight from their definition; test infrastructure only."""
import numpy as np

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step, relative


def steps_of(cols):
    return -(-cols // 128)


def _blocks(x):
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    pad = np.zeros((rows, steps_of(cols) * 128))
    pad[:, :cols] = x
    return pad.reshape(rows, -1, 32)


def _exponents(b, top):
    m = np.abs(b).max(axis=2) if b.shape[1] else np.zeros(b.shape[:2])
    bad = ~np.isfinite(m)
    m = np.where(bad | (m == 0), 1.0, m)
    e = np.frexp(m)[1] - 1 - top  # floor(log2)
    e = np.where(np.abs(b).max(axis=2, initial=0) == 0, -127, np.maximum(e, -127))
    return e, bad


def mx4_quantize(x):
    """(codes uint8 [rows, steps * 64], scales uint8 [rows, steps * 4])"""
    b = _blocks(x)
    e, bad = _exponents(b, 2)
    v = np.where(bad[:, :, None], 0.0, b)
    a = np.abs(v) / np.exp2(e.astype(np.float64))[:, :, None]
    code = np.zeros(a.shape, dtype=np.uint8)
    for i in range(7):  # past the middle of codes i and i + 1, or on it where i + 1 is even
        mid = (GRID[i] + GRID[i + 1]) / 2
        code[(a > mid) | ((a == mid) & (i % 2 == 1))] = i + 1
    code |= (np.signbit(v) << 3).astype(np.uint8)
    code = code.reshape(b.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), np.where(bad, 255, e + 127).astype(np.uint8)


def mx4_decode(codes, scales, cols):
    codes = np.asarray(codes)
    full = np.empty((codes.shape[0], codes.shape[1] * 2), dtype=np.uint8)
    full[:, 0::2], full[:, 1::2] = codes & 15, codes >> 4
    v = GRID[full & 7] * np.where(full & 8, -1.0, 1.0)
    return _scaled(v, scales)[:, :cols]


def act8_quantize(x):
    b = _blocks(x)
    e, bad = _exponents(b, 6)
    v = np.where(bad[:, :, None], 0.0, b)
    q = np.clip(np.rint(v / np.exp2(e.astype(np.float64))[:, :, None]), -127, 127).astype(np.int8)
    return q.reshape(b.shape[0], -1), np.where(bad, 255, e + 127).astype(np.uint8)


def act8_decode(codes, scales, cols):
    return _scaled(np.asarray(codes).astype(np.float64), scales)[:, :cols]


def _scaled(v, scales):
    s = np.asarray(scales).astype(np.float64)
    s = np.where(s == 255, np.nan, np.exp2(s - 127))
    return v * np.repeat(s, 32, axis=1)


def _normal(x):
    from scipy.special import ndtr
    return ndtr(x)


def activation(x, fn):
    x = np.asarray(x, dtype=np.float64)
    if fn == "gelu":
        return x * _normal(x)
    return x / (1 + np.exp(-x))


def slope(x, fn):
    x = np.asarray(x, dtype=np.float64)
    if fn == "gelu":
        return _normal(x) + x * np.exp(-x * x / 2) / np.sqrt(2 * np.pi)
    g = 1 / (1 + np.exp(-x))
    return g * (1 + x * (1 - g))
