"""Shared by the GPU tests of the microscaled operators: inputs, packing through numpy, bounds."""
import numpy as np
import torch

import mx_ref as ref

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def name(dtype):
    return str(dtype).replace("torch.", "")


def half_step(dtype):
    return ref.U[name(dtype)]


def f64(t):
    return t.detach().double().cpu().numpy()


def values(seed, rows, cols, dtype, scale=1.0):
    """Normal numbers over several powers of two with large channels, zero rows and zero blocks."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * scale
    x *= torch.exp2(torch.randint(-6, 3, (rows, 1), generator=g).float())
    x[:, ::17] *= 20
    if rows > 3:
        x[rows // 2] = 0
    if cols > 70:
        x[0, 32:64] = 0
    return x.to(dtype).cuda()


def widened(t, left=3, right=5):
    """The same matrix as a column range of a wider one, which is filled with NaN around it."""
    wide = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), dtype=t.dtype, device=t.device)
    view = wide[:, left:left + t.shape[1]]
    view.copy_(t)
    return view, wide


def untouched(wide, left, cols):
    w = wide.clone()
    w[:, left:left + cols] = float("nan")
    return bool(torch.isnan(w).all())


def packed4(x):
    """mx4 codes and scales on the GPU of what numpy quantizes, and the values they stand for."""
    c, s = ref.mx4_quantize(f64(x) if isinstance(x, torch.Tensor) else x)
    return torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), ref.mx4_decode(c, s, x.shape[1])


def packed8(x):
    c, s = ref.act8_quantize(f64(x))
    return torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda(), ref.act8_decode(c, s, x.shape[1])


def matmul64(a, b):
    """a @ b of numpy matrices in 64 bits, on the GPU."""
    return (torch.from_numpy(np.ascontiguousarray(a)).cuda() @ torch.from_numpy(np.ascontiguousarray(b)).cuda()).cpu().numpy()


def assert_within(got, want, bound, what=""):
    got = f64(got) if isinstance(got, torch.Tensor) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = np.abs(got - want) - bound
    assert not np.isnan(got).any(), f"{what}: NaN"
    if off.size and off.max() > 0:
        at = np.unravel_index(off.argmax(), off.shape)
        raise AssertionError(f"{what}: at {at}: got {got[at]!r} want {want[at]!r}, off by {abs(got[at] - want[at]):.3g}, "
                             f"bound {np.broadcast_to(bound, want.shape)[at]:.3g}; {int((off > 0).sum())} of {off.size} beyond")
