"""Arguments of the layers: biases that are not contiguous, and what is refused by name."""
import pytest
import torch

from mx_gpu import values
from necklace_amd.frmwrk.pytorch import ptmx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
def test_biases_that_are_not_contiguous(layer):
    x, w = values(1, 40, 100, torch.float32), values(2, 30, 100, torch.float32)
    table = torch.randn(30, 4, device="cuda")
    for bias in (table[:, 1], torch.ones(1, device="cuda").expand(30)):
        b = bias.detach().requires_grad_()
        c = bias.detach().contiguous().requires_grad_()
        y, want = layer(x, w, b), layer(x, w, c)
        assert torch.equal(y, want)
        assert torch.equal(torch.autograd.grad(y.sum(), b)[0], torch.autograd.grad(want.sum(), c)[0])
        with torch.no_grad():
            served = ptmx.Mx4Weight(w)
            assert torch.equal(served.linear(x, bias), served.linear(x, bias.contiguous()))


def test_refusals_by_name():
    w = torch.zeros(5, 8, device="cuda")
    for bad, error in (([1.0], TypeError), (w.cpu(), TypeError), (w.double(), TypeError), (w[0], ValueError), (w[None], ValueError),
                       (None, TypeError)):
        with pytest.raises(error, match="weight"):
            ptmx.Mx4Weight(bad)
    served = ptmx.Mx4Weight(w)
    with torch.no_grad():
        for bad in ([1.0], torch.zeros(4, 8), None):
            with pytest.raises(TypeError, match="x: expected a GPU tensor"):
                served.linear(bad)
        with pytest.raises(TypeError, match="bias"):
            served.linear(torch.zeros(4, 8, device="cuda"), [0.0] * 5)
        with pytest.raises(ValueError, match="bias"):
            served.linear(torch.zeros(4, 8, device="cuda"), torch.zeros(4, device="cuda"))
    for layer in (ptmx.act8_linear, ptmx.mx4_linear):
        with pytest.raises(TypeError, match="x: expected a torch tensor"):
            layer(None, w)
        with pytest.raises(TypeError, match="weight: expected a torch tensor"):
            layer(w, None)
    with pytest.raises(TypeError, match="x: expected a torch tensor"):
        ptmx.act8_act([1.0], "gelu")
