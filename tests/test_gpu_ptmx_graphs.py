"""Layers captured into a graph, replayed with eager work between, every replay compared; bias gradients of frozen layers."""
import pytest
import torch

from mx_gpu import DTYPES, name, values
from necklace_amd.cuda import mx
from necklace_amd.frmwrk.pytorch import ptmx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
@pytest.mark.parametrize("t,n", [(150, 60), (20000, 64), (3000, 1000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_bias_gradient_of_a_frozen_layer_in_a_graph(layer, t, n, dtype):
    x = values(1, t, 48, dtype, 0.1)
    w = values(2, n, 48, dtype, 0.1)
    b = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    dy = torch.zeros(t, n, dtype=dtype, device="cuda")

    def step():
        return torch.autograd.grad(layer(x, w, b), b, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(5):
        dy.copy_(values(seed + 3, t, n, dtype, 0.1))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, step())
        # t / 4 + 16 + 257 roundings of a sum's part at most, and one to the type
        want, mags = dy.double().sum(0), dy.double().abs().sum(0)
        bound = (t / 4 + 273) * 2.0 ** -24 * mags
        bound = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound) + 2.0 ** -25
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
@pytest.mark.parametrize("t,n,k", [(150, 60, 100), (20000, 64, 48), (3000, 1000, 520), (32, 64, 8192), (32, 8192, 64), (1, 4096, 4096)])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_a_layer_with_its_activation_in_a_graph(layer, t, n, k, dtype):
    """Result and all gradients of every replay against the eager calls, which run between the replays."""
    x = values(1, t, k, dtype, 0.1).requires_grad_()
    w = values(2, n, k, dtype, 0.1).requires_grad_()
    b = torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    dy = values(3, t, n, dtype, 0.1)

    def step():
        y = ptmx.act8_act(layer(x, w, b), "gelu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in range(5):
        dy.copy_(values(seed + 3, t, n, dtype, 0.1))
        with torch.no_grad():
            x.copy_(values(seed + 9, t, k, dtype, 0.1))
        g.replay()
        torch.cuda.synchronize()
        for what, a, e in zip(("y", "dx", "dw", "db"), got, step()):
            assert torch.equal(a, e), (what, seed)


@pytest.mark.parametrize("shape", [(300, 1), (7, 3), (1, 1000), (40, 129), (2000, 257), (70000, 4), (513, 5000)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_bias_gradient_alone(shape, dtype):
    """db without columns of x: sums of strided rows, onto what is there, NaN and infinity in their columns alone."""
    t, n = shape
    wide = torch.full((t, n + 3), float("nan"), dtype=dtype, device="cuda")
    dy = wide[:, 1:1 + n]
    dy.copy_(values(t, t, n, dtype, 0.1))
    c, s = mx.act8_empty(t, 0)
    none, db = torch.empty(n, 0, device="cuda"), torch.full((n,), float("nan"), device="cuda")
    mx.cu_fn_act8_wgrad_e(none, dy, c, s, DB=db)
    want, mags = dy.double().sum(0), dy.double().abs().sum(0)
    bound = (t / 4 + 273) * 2.0 ** -24 * mags
    assert bool(((db.double() - want).abs() <= bound).all())
    twice = db.clone()
    mx.cu_fn_act8_wgrad_e(none, dy, c, s, DB=twice, accumulate=True)
    assert bool(((twice.double() - 2 * want).abs() <= 2 * bound + 2.0 ** -23 * want.abs()).all())
    dy[t - 1, 0], dy[0, n - 1] = float("inf"), float("nan")
    bad = db.clone()
    mx.cu_fn_act8_wgrad_e(none, dy, c, s, DB=bad)
    assert bool(torch.isnan(bad[n - 1])) and (n == 1 or float(bad[0]) == float("inf"))
    assert torch.equal(bad[1:n - 1], db[1:n - 1])


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
def test_a_frozen_layer_without_outputs(layer):
    x, w = torch.randn(5, 48, device="cuda"), torch.randn(0, 48, device="cuda")
    b = torch.randn(0, device="cuda", requires_grad=True)
    y = layer(x, w, b)
    assert torch.autograd.grad(y.sum(), b)[0].shape == (0,)


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
def test_layers_on_another_stream(layer):
    """Forward and backward behind slow work of a side stream: results and gradients as on the default one."""
    x = values(1, 3000, 200, torch.bfloat16, 0.1)
    w = values(2, 300, 200, torch.bfloat16, 0.1).requires_grad_()
    b = torch.zeros(300, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    dy = values(3, 3000, 300, torch.bfloat16, 0.1)

    def step(x):
        x = x.detach().requires_grad_()
        y = ptmx.act8_act(layer(x, w, b), "silu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    want = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(x)
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = (big @ big).clamp(-1, 1)
        late.copy_(x)
        late += (big[0, 0] * 0).to(x.dtype)
        got = step(late)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
