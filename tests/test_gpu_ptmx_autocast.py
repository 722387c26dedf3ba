"""Layers in mixed precision: bf16 activations beside fp32 weights in an autocast region."""
import pytest
import torch

from necklace_amd.frmwrk.pytorch import ptmx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("types", [(0, 1, 1), (1, 0, 0), (0, 0, 1), (0, 1, 0)], ids=str)
def test_different_types_are_cast_to_the_region_s(layer, dtype, types):
    """types: which of x, weight and bias are fp32; the others are of the region's type."""
    g = torch.Generator(device="cuda").manual_seed(1)
    shapes = [(5, 30, 100), (70, 100), (70,)]
    made = [torch.randn(s, device="cuda", generator=g) * 0.1 for s in shapes]
    args = [t.to(torch.float32 if wide else dtype).requires_grad_() for t, wide in zip(made, types)]
    cast = [t.detach().to(dtype).requires_grad_() for t in args]
    dy = torch.randn(5, 30, 70, device="cuda", generator=g).to(dtype)
    with torch.autocast("cuda", dtype=dtype):
        y = layer(*args)
    assert y.dtype == dtype
    want = layer(*cast)
    assert torch.equal(y, want)
    for a, b, t in zip(torch.autograd.grad(y, args, dy), torch.autograd.grad(want, cast, dy), args):
        assert a.dtype == t.dtype and torch.equal(a, b.to(t.dtype))


def test_a_model_of_torch_s_and_these_layers():
    """torch's linear layer hands on bf16; its fp32 weights and theirs train side by side."""
    torch.manual_seed(3)
    first = torch.nn.Linear(64, 128, device="cuda")
    w, b = torch.nn.Parameter(torch.randn(32, 128, device="cuda") * 0.1), torch.nn.Parameter(torch.zeros(32, device="cuda"))
    x = torch.randn(40, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ptmx.act8_linear(ptmx.act8_act(first(x), "gelu"), w, b)
        assert y.dtype == torch.bfloat16
        served = ptmx.Mx4Weight(w)
        with torch.no_grad():
            z = served.linear(first(x), b)
            assert z.dtype == torch.bfloat16 and torch.equal(z, served.linear(first(x), b.bfloat16()))
    y.float().square().mean().backward()
    assert all(p.grad is not None and p.grad.dtype == torch.float32 for p in (first.weight, first.bias, w, b))


def test_without_autocast_different_types_are_refused():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    for layer in (ptmx.act8_linear, ptmx.mx4_linear):
        with pytest.raises(TypeError, match="weight is"):
            layer(x.bfloat16(), w)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            with pytest.raises(TypeError, match="weight"):
                layer(x, w.double())
            with pytest.raises(TypeError, match="tensor"):
                layer(x, w, [0.0] * 5)
    with pytest.raises(TypeError, match="bias"), torch.no_grad():
        ptmx.Mx4Weight(w).linear(x.bfloat16(), torch.zeros(5, device="cuda"))
