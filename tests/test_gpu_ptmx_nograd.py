"""The layers where no gradient can be asked for: the same results, and nothing is kept."""
import pytest
import torch

from mx_gpu import DTYPES, name, untouched, values, widened
from necklace_amd.cuda import mx
from necklace_amd.frmwrk.pytorch import ptmx

pytestmark = pytest.mark.gpu


@pytest.fixture
def checkpoints(monkeypatch):
    """Shapes of the checkpoints that are laid out."""
    made = []
    original = mx.act8_empty

    def counted(rows, cols, device="cuda"):
        made.append((rows, cols))
        return original(rows, cols, device=device)

    monkeypatch.setattr(mx, "act8_empty", counted)
    return made


def calls():
    x = values(1, 150, 100, torch.bfloat16, 0.1).requires_grad_()
    w = values(2, 60, 100, torch.bfloat16, 0.1).requires_grad_()
    b = torch.randn(60, device="cuda").bfloat16().requires_grad_()
    return {"act8_linear": lambda: ptmx.act8_linear(x, w, b), "mx4_linear": lambda: ptmx.mx4_linear(x, w, b),
            "gelu": lambda: ptmx.act8_act(x, "gelu"), "silu": lambda: ptmx.act8_act(x, "silu")}


@pytest.mark.parametrize("which", ["act8_linear", "mx4_linear", "gelu", "silu"])
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_nothing_is_kept_without_gradients(checkpoints, which, mode):
    call = calls()[which]
    want = call()
    assert checkpoints == [(150, 100)] and want.requires_grad
    checkpoints.clear()
    with mode():
        got = call()
    assert checkpoints == [] and not got.requires_grad
    assert torch.equal(got, want)


def test_nothing_is_kept_for_inputs_that_need_no_gradient(checkpoints):
    x = values(1, 150, 100, torch.bfloat16, 0.1)
    w = values(2, 60, 100, torch.bfloat16, 0.1)
    for call in (lambda: ptmx.act8_linear(x, w), lambda: ptmx.mx4_linear(x, w), lambda: ptmx.act8_act(x, "gelu")):
        call()
    w.requires_grad_()
    ptmx.act8_act(x, "gelu")
    assert checkpoints == []
    ptmx.act8_linear(x, w)
    assert checkpoints == [(150, 100)]


@pytest.mark.parametrize("fn", ["gelu", "silu"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (257, 64), (33, 1000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_an_activation_alone_has_the_same_bits(rows, cols, dtype, fn):
    x, _ = widened(values(rows, rows, cols, dtype), 1, 4)
    x[rows // 2, cols - 1] = float("nan")
    c, s = mx.act8_empty(rows, cols)
    want, (got, wide) = torch.empty(rows, cols, dtype=dtype, device="cuda"), widened(torch.zeros(rows, cols, dtype=dtype, device="cuda"))
    mx.cu_fn_act8_save_e(x, c, s, Y=want, fn=fn)
    mx.cu_fn_act8_save_e(x, None, None, Y=got, fn=fn)
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)) and torch.equal(got.isnan(), want.isnan())
    assert untouched(wide, 3, cols)
    z = x.clone()
    mx.cu_fn_act8_save_e(z, None, None, Y=z, fn=fn)
    assert torch.equal(z.nan_to_num(), want.nan_to_num())


def test_half_a_checkpoint_is_refused():
    x = torch.zeros(4, 300, device="cuda")
    c, s = mx.act8_empty(4, 300)
    for pair in ((c, None), (None, s)):
        with pytest.raises(TypeError, match="torch tensor"):
            mx.cu_fn_act8_save_e(x, *pair, Y=torch.empty_like(x), fn="gelu")
    with pytest.raises(TypeError, match="torch tensor"):
        mx.cu_fn_act8_save_e(x, None, None)


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
def test_a_weight_that_no_gradient_reads_may_change(layer):
    """Only the input's gradient reads the weight: without it the weight may be updated before the backward pass, as with
    torch's linear layer; with it the change is noticed."""
    x, w = values(1, 50, 100, torch.float32), values(2, 30, 100, torch.float32).requires_grad_()
    dy = values(3, 50, 30, torch.float32)
    want, = torch.autograd.grad(layer(x, w), w, dy)
    y = layer(x, w)
    with torch.no_grad():
        w.add_(1)
    got, = torch.autograd.grad(y, w, dy)
    assert torch.equal(got, want)
    y = layer(x.requires_grad_(), w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, (x, w), dy)
