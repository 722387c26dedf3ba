"""Layers whose stored tensors are microscaled: what a training step keeps between forward and backward, and what a
product reads, in 8 and 4 bits.  Beside ptcomp (which packs the gradients a step sends), on the kernels of
necklace_amd.cuda.mx.

    act8_linear(x, weight, bias)   y = x W^T + b by torch; x is kept in 8 bits and the weight gradient read from it
    act8_act(x, fn)                y = fn(x), "gelu" or "silu"; x is kept in 8 bits and the gradient read from it
    mx4_linear(x, weight, bias)    y = mx4(x) mx4(W)^T + b; backward dx = mx4(dy) mx4(W^T)^T, dW as in act8_linear:
                                   the rounding is treated as the identity (straight through)
    Mx4Weight(weight)              the codes alone, laid out once: .linear(x, bias) for serving

Nothing is kept where no gradient can ask for it (without gradients enabled, or with inputs that need none).

x is float32, bfloat16 or float16 on the GPU, [..., in]; weight [out, in] and bias [out] of the same type.  In an
autocast region equal types stay as they are; different ones (bf16 activations beside fp32 weights) are cast to the region's
type.  Gradients have their tensor's type; the weight gradient is summed in fp32 whatever that is.  The calls run on torch's
current stream and can be captured into a graph.  A backward pass that is captured has to be the first use of its leaves'
gradients on that stream (torch's own rule): take them with `torch.autograd.grad`, or let no eager graph of the same
leaves live during the capture.  Second derivatives are not available.
"""
import torch
from torch.autograd.function import once_differentiable

from ...cuda import mx


def _as_given():
    """Types stay what the caller brought, inside an autocast region too."""
    return torch.autocast("cuda", enabled=False)


def _rows(t):
    """`t` where its strides are rows of neighbouring columns, else a contiguous copy (an expanded gradient)."""
    return t if mx.row_stride(t) is not None else t.contiguous()


def _one_type(x, weight, bias):
    """In an autocast region tensors of different types are cast to its type, as in torch's own linear layer; the casts
    carry the gradients back to each tensor's own type."""
    tensors = [x, weight] + ([] if bias is None else [bias])
    if torch.is_autocast_enabled("cuda") and all(isinstance(t, torch.Tensor) and t.dtype in mx._TYPES for t in tensors) \
            and any(t.dtype != x.dtype for t in tensors):
        dtype = torch.get_autocast_dtype("cuda")
        return tuple(t if t is None else t.to(dtype) for t in (x, weight, bias))
    return x, weight, bias


def _check_tensor(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if t.dtype not in mx._TYPES or not t.is_cuda:
        raise TypeError(f"{name}: expected a float32, bfloat16 or float16 GPU tensor, got {t.dtype} on {t.device}")


def _check(x, *weight_and_bias):
    _check_tensor("x", x)
    if x.dim() < 1:
        raise ValueError("x: expected at least 1 dimension")
    if not weight_and_bias:
        return
    weight, bias = weight_and_bias
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None and name == "bias":
            continue
        _check_tensor(name, t)
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias {tuple(bias.shape)} does not fit weight {tuple(weight.shape)}")


def _save(x):
    x = _rows(x)
    rows, cols = mx.shape2(x)
    c, s = mx.act8_empty(rows, cols, device=x.device)
    mx.cu_fn_act8_save_e(x, c, s, sync=False)
    return c, s


def _column_sums(dy):
    """fp32 sums of dy's columns: the weight gradient's bias alone.  (torch's sum clears its scratch memory by a graph node
    that gives wrong sums when a captured graph is replayed.)"""
    rows, n = mx.shape2(dy)
    c, s = mx.act8_empty(rows, 0, device=dy.device)
    db = torch.empty(n, dtype=torch.float32, device=dy.device)
    mx.cu_fn_act8_wgrad_e(db.new_empty(n, 0), dy, c, s, DB=db, sync=False)
    return db


def _weight_grads(dy, c, s, weight_like, need_w, need_b):
    """Gradients of weight and bias from the checkpoint, in the weight's type."""
    if not need_w:
        return None, (_column_sums(dy).to(dy.dtype) if need_b else None)
    n, k = weight_like
    dw = torch.empty(n, k, dtype=torch.float32, device=dy.device)
    db = torch.empty(n, dtype=torch.float32, device=dy.device) if need_b else None
    mx.cu_fn_act8_wgrad_e(dw, dy, c, s, DB=db, sync=False)
    return dw.to(dy.dtype), db.to(dy.dtype) if need_b else None


def _keep(ctx, x, weight, keep):
    """What backward reads: the weight for the input's gradient, the checkpoint of x for the weight's."""
    ctx.weight_shape = weight.shape
    ctx.saved_w, ctx.saved_x = keep and ctx.needs_input_grad[0], keep and ctx.needs_input_grad[1]
    ctx.save_for_backward(*((weight,) if ctx.saved_w else ()), *(_save(x) if ctx.saved_x else ()))


def _kept(ctx):
    """(weight, codes, scales), None where not kept."""
    kept = ctx.saved_tensors
    return (kept[0] if ctx.saved_w else None,) + (kept[-2:] if ctx.saved_x else (None, None))


class _Act8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, keep):
        _keep(ctx, x, weight, keep)
        with _as_given():
            return torch.nn.functional.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, c, s = _kept(ctx)
        dy = _rows(dy)
        with _as_given():
            dx = dy @ weight if ctx.needs_input_grad[0] else None
        dw, db = _weight_grads(dy, c, s, ctx.weight_shape, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return dx, dw, db, None


class _Act8Act(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, fn, keep):
        x = _rows(x)
        c = s = None
        if keep and ctx.needs_input_grad[0]:
            c, s = mx.act8_empty(*mx.shape2(x), device=x.device)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        mx.cu_fn_act8_save_e(x, c, s, Y=y, fn=fn, sync=False)
        ctx.save_for_backward(c, s)
        ctx.fn = fn
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        c, s = ctx.saved_tensors
        dy = _rows(dy)
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dy.device)
        mx.cu_fn_act8_grad_e(dx, dy, c, s, ctx.fn, sync=False)
        return dx, None, None


class _Mx4Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, keep):
        _keep(ctx, x, weight, keep)
        return Mx4Weight(weight).linear(x, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        weight, c, s = _kept(ctx)
        dy = _rows(dy)
        dx = None
        if ctx.needs_input_grad[0]:
            dx = Mx4Weight(weight, transpose=True).linear(dy)
        dw, db = _weight_grads(dy, c, s, ctx.weight_shape, ctx.needs_input_grad[1], ctx.needs_input_grad[2])
        return dx, dw, db, None


def act8_linear(x, weight, bias=None):
    """torch.nn.functional.linear that keeps x in 8 bits (a quarter of fp32, half of 16 bits) for the weight gradient."""
    x, weight, bias = _one_type(x, weight, bias)
    _check(x, weight, bias)
    return _Act8Linear.apply(x, weight, bias, torch.is_grad_enabled())


def act8_act(x, fn):
    """fn(x) ("gelu": x Phi(x), "silu": x / (1 + e^-x)) that keeps x in 8 bits for its gradient."""
    _check(x)
    mx._fn_code(fn, False)
    return _Act8Act.apply(x, fn, torch.is_grad_enabled())


def mx4_linear(x, weight, bias=None):
    """A linear layer whose products run on 4-bit operands, with gradients; the weight is laid out anew in every pass."""
    x, weight, bias = _one_type(x, weight, bias)
    _check(x, weight, bias)
    return _Mx4Linear.apply(x, weight, bias, torch.is_grad_enabled())


class Mx4Weight:
    """The mx4 codes of a weight [out, in] (of its transpose with ``transpose=True``): 4.25 bits an element."""

    def __init__(self, weight, transpose=False):
        _check_tensor("weight", weight)
        if weight.dim() != 2:
            raise ValueError(f"weight: expected 2 dimensions, got {weight.dim()}")
        w = _rows(weight.detach())
        n, k = w.shape
        self.shape = (k, n) if transpose else (n, k)
        self.codes, self.scales = mx.mx4_empty(*self.shape, device=w.device)
        mx.cu_fn_mx4_quantize_e(w, self.codes, self.scales, transpose=transpose, sync=False)

    def linear(self, x, bias=None):
        """mx4(x) W^T (+ bias), [..., in] -> [..., out]; for use without gradients."""
        if not (isinstance(x, torch.Tensor) and x.is_cuda):
            raise TypeError("x: expected a GPU tensor")
        if bias is not None:
            if not isinstance(bias, torch.Tensor):
                raise TypeError(f"bias: expected a torch tensor, got {type(bias).__name__}")
            if not bias.is_contiguous():
                bias = bias.contiguous()
            if bias.dtype != x.dtype and torch.is_autocast_enabled("cuda"):
                bias = bias.to(x.dtype)
        if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError("Mx4Weight.linear has no gradient: use mx4_linear, or torch.no_grad()")
        if x.dim() < 1 or x.shape[-1] != self.shape[1]:
            raise ValueError(f"x {tuple(x.shape)} does not fit the weight {self.shape}")
        x = _rows(x)
        y = torch.empty(*x.shape[:-1], self.shape[0], dtype=x.dtype, device=x.device)
        mx.cu_fn_mx4_linear_e(y, x, self.codes, self.scales, bias=bias, sync=False)
        return y
