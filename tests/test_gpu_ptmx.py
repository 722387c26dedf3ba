"""The microscaled layers and their calls as a program uses them: gradients, streams, threads, graphs, a training step
whose gradients the 2-bit compressor packs."""
import threading

import numpy as np
import pytest
import torch

import mx_ref as ref
from mx_gpu import DTYPES, assert_within, f64, half_step, matmul64, name, packed4, packed8, values
from necklace_amd.cuda import mx
from necklace_amd.frmwrk.pytorch import ptcomp, ptmx
from test_gpu_act8 import slope_bound, wgrad_bounds
from test_gpu_mx4 import product_bound

pytestmark = pytest.mark.gpu


def saved8(x):
    return ref.act8_decode(*ref.act8_quantize(f64(x)), x.shape[-1])


def coded4(x):
    return ref.mx4_decode(*ref.mx4_quantize(f64(x)), x.shape[-1])


def to_type(bound, want, dtype):
    """A bound of an fp32 result that is rounded once more to a gradient's type."""
    return bound + half_step(dtype) * (np.abs(want) + bound) + (2.0 ** -25 if dtype == torch.float16 else 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_act8_linear(dtype):
    x = values(1, 6 * 50, 100, dtype, 0.1).view(6, 50, 100).requires_grad_()
    w = values(2, 70, 100, dtype, 0.1).requires_grad_()
    b = torch.randn(70, device="cuda").to(dtype).requires_grad_()
    dy = values(3, 300, 70, dtype, 0.1).view(6, 50, 70)
    y = ptmx.act8_linear(x, w, b)
    assert torch.equal(y, torch.nn.functional.linear(x, w, b))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert torch.equal(dx, dy @ w)
    d64, x64 = f64(dy).reshape(300, 70), saved8(x.detach().view(300, 100))
    bound_w, bound_b = wgrad_bounds(d64, x64, 300, dtype)
    want = matmul64(d64.T, x64)
    assert_within(dw, want, to_type(bound_w, want, dtype), "dw")
    assert_within(db, d64.sum(0), to_type(bound_b, d64.sum(0), dtype), "db")


@pytest.mark.parametrize("fn", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=name)
def test_act8_act(dtype, fn):
    x = values(1, 60, 100, dtype, 0.3).view(3, 20, 100).requires_grad_()
    dy = values(2, 60, 100, dtype).view(3, 20, 100)
    y = ptmx.act8_act(x, fn)
    assert y.shape == x.shape and y.dtype == dtype
    dx, = torch.autograd.grad(y, x, dy)
    x64, d64 = saved8(x.detach().view(60, 100)), f64(dy).reshape(60, 100)
    want = d64 * ref.slope(x64, fn)
    assert_within(f64(dx).reshape(60, 100), want, slope_bound(x64, d64, want, fn, dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=name)
@pytest.mark.parametrize("rows", [2, 300])
def test_mx4_linear(dtype, rows):
    x = values(1, rows, 100, dtype, 0.1).requires_grad_()
    w = values(2, 70, 100, dtype, 0.1).requires_grad_()
    b = torch.randn(70, device="cuda").to(dtype).requires_grad_()
    dy = values(3, rows, 70, dtype, 0.1)
    y = ptmx.mx4_linear(x, w, b)
    a64, w64 = coded4(x), coded4(w)
    want = matmul64(a64, w64.T) + f64(b)
    assert_within(y, want, product_bound(a64, w64, want, 100, dtype, f64(b)), "y")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    d4, wt = coded4(dy), coded4(w.detach().t())
    want = matmul64(d4, wt.T)
    assert_within(dx, want, product_bound(d4, wt, want, 70, dtype), "dx")
    d64, x64 = f64(dy), saved8(x)
    bound_w, bound_b = wgrad_bounds(d64, x64, rows, dtype)
    want = matmul64(d64.T, x64)
    assert_within(dw, want, to_type(bound_w, want, dtype), "dw")
    assert_within(db, d64.sum(0), to_type(bound_b, d64.sum(0), dtype), "db")


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_only_the_gradients_that_are_asked_for(layer, need):
    make = lambda: [values(1, 40, 64, torch.float32).requires_grad_(), values(2, 30, 64, torch.float32).requires_grad_(),  # noqa: E731
                    torch.ones(30, device="cuda").requires_grad_()]
    dy = values(3, 40, 30, torch.float32)
    full = make()
    layer(*full).backward(dy)
    some = make()
    for t, n in zip(some, need):
        t.requires_grad_(bool(n))
    layer(*some).backward(dy)
    for a, b, n in zip(full, some, need):
        if not n:
            assert b.grad is None
        elif a is full[2]:  # without the weight's gradient the bias is summed by torch
            assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=1e-4)
        else:
            assert torch.equal(a.grad, b.grad)


def test_expanded_gradients_and_strided_inputs():
    base = values(1, 40, 200, torch.float32).t()  # [200, 40] with the columns apart
    for x in (base, values(1, 40, 200, torch.float32)[:, 30:130]):
        x = x.detach().requires_grad_()
        w = values(2, 30, x.shape[1], torch.float32).requires_grad_()
        ptmx.mx4_linear(x, w).sum().backward()  # dy is one number with strides 0
        y = x.detach().contiguous().requires_grad_()
        v = w.detach().clone().requires_grad_()
        out = ptmx.mx4_linear(y, v)
        out.backward(torch.ones_like(out))
        assert torch.equal(x.grad, y.grad) and torch.equal(w.grad, v.grad)
        x.grad = y.grad = None
        ptmx.act8_act(x, "gelu").sum().backward()
        out = ptmx.act8_act(y, "gelu")
        out.backward(torch.ones_like(out))
        assert torch.equal(x.grad, y.grad)


def test_checkpoints_take_a_quarter_of_fp32():
    x = torch.randn(4096, 1024, device="cuda", requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ptmx.act8_act(x, "silu")
    held = torch.cuda.memory_allocated() - before - y.numel() * 4
    assert held <= x.numel() * 33 / 32 + 4096
    del y


def test_refusals():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(5, 8, device="cuda")
    for layer in (ptmx.act8_linear, ptmx.mx4_linear):
        with pytest.raises(TypeError, match="weight is"):
            layer(x, w.bfloat16())
        with pytest.raises(ValueError, match="weight"):
            layer(x, w[:, :7])
        with pytest.raises(ValueError, match="bias"):
            layer(x, w, torch.zeros(4, device="cuda"))
        with pytest.raises(TypeError, match="GPU"):
            layer(x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="fn"):
        ptmx.act8_act(x, "relu")
    with pytest.raises(RuntimeError, match="no gradient"):
        ptmx.Mx4Weight(w).linear(x.requires_grad_())
    with torch.no_grad():
        assert ptmx.Mx4Weight(w).linear(x).shape == (4, 5)
        with pytest.raises(ValueError, match="fit"):
            ptmx.Mx4Weight(w).linear(x[:, :5])
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(ptmx.act8_act(x, "gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_autocast_does_not_change_types():
    x, w = torch.randn(4, 8, device="cuda", requires_grad=True), torch.randn(5, 8, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for layer in (ptmx.act8_linear, ptmx.mx4_linear):
            y = layer(x, w)
            assert y.dtype == torch.float32
            dx, dw = torch.autograd.grad(y.sum(), (x, w))
            assert dx.dtype == dw.dtype == torch.float32


# ---- together

def mlp(x, w1, b1, w2, mx4):
    layer = ptmx.mx4_linear if mx4 else ptmx.act8_linear
    return layer(ptmx.act8_act(layer(x, w1, b1), "gelu"), w2)


def leaves(dtype=torch.float32):
    g = torch.Generator().manual_seed(5)
    shapes = [(200, 100), (200,), (60, 200)]
    return [(torch.randn(*s, generator=g) * 0.1).to(dtype).cuda().requires_grad_() for s in shapes]


@pytest.mark.parametrize("mx4", [False, True], ids=["act8", "mx4"])
def test_a_training_step_whose_gradients_the_compressor_packs(mx4):
    params = leaves()
    gc = ptcomp.GradCompressor(params, kn=1, thrd=0.05, size_threshold=100)
    owed = [torch.zeros_like(p) for p in params]
    for step in range(3):
        x = values(step, 150, 100, torch.float32, 0.1)
        for p in params:
            p.grad = None
        loss = mlp(x, *params, mx4).square().mean()
        loss.backward()
        # the last layer's gradient by the formula
        with torch.no_grad():
            h = mlp_hidden(x, params, mx4)
            y = mlp(x, *params, mx4)
        d64, h64 = f64(2 * y / y.numel()), saved8(h)
        want = matmul64(d64.T, h64)
        bound, _ = wgrad_bounds(d64, h64, 150, torch.float32)
        assert_within(params[2].grad, want, bound + 2.0 ** -22 * matmul64(np.abs(d64).T, np.abs(h64)))
        grads = [p.grad.clone() for p in params]
        gc.compress([p.grad for p in params])
        outs = [torch.empty_like(p) for p in params]
        gc.decompress_sum(outs)
        for i, p in enumerate(params):  # what was sent and what is kept make up what was owed
            owed[i] = owed[i] + grads[i]
            left = gc.grd_resi[i].view_as(p)
            assert torch.equal(torch.where(outs[i] == 0, owed[i], owed[i] - outs[i]), left)
            owed[i] = left.clone()
            with torch.no_grad():
                p -= 0.1 * outs[i]


def mlp_hidden(x, params, mx4):
    layer = ptmx.mx4_linear if mx4 else ptmx.act8_linear
    return ptmx.act8_act(layer(x, params[0], params[1]), "gelu")


def test_serving_one_token_after_a_prompt():
    w = values(1, 300, 200, torch.bfloat16, 0.1)
    with torch.no_grad():
        packed = ptmx.Mx4Weight(w)
        x = values(2, 130, 200, torch.bfloat16)
        whole = packed.linear(x)
        a, b = coded4(x), coded4(w)
        for i in (0, 5, 129):
            one = packed.linear(x[i:i + 1])
            want = matmul64(a[i:i + 1], b.T)
            bound = product_bound(a[i:i + 1], b, want, 200, torch.bfloat16)
            assert_within(one, want, bound)
            assert_within(whole[i:i + 1], want, bound)


# ---- streams, threads, graphs

def problem(seed, t=3000, n=70, k=130):
    c, s, _ = packed8(values(seed, t, k, torch.bfloat16))
    dy = values(seed + 1, t, n, torch.bfloat16)
    cb, sb, _ = packed4(f64(values(seed + 2, n, k, torch.float32)))
    x = values(seed + 3, 100, k, torch.bfloat16)
    return dict(c=c, s=s, dy=dy, cb=cb, sb=sb, x=x)


def run(p, stream=None, sync=False):
    dw, db = torch.empty(70, 130, device="cuda"), torch.empty(70, device="cuda")
    y = torch.empty(100, 70, dtype=torch.bfloat16, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, p["dy"], p["c"], p["s"], DB=db, stream=stream, sync=sync)
    mx.cu_fn_mx4_linear_e(y, p["x"], p["cb"], p["sb"], stream=stream, sync=sync)
    return dw, db, y


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_streams_and_raw_handles():
    assert mx.act8_wgrad_workspace(torch.bfloat16, 3000, 70, 130) > 0 and mx.mx4_linear_workspace(100, 70, 130) > 0
    p = problem(1)
    want = run(p)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream, torch.cuda.current_stream().cuda_stream):
        got = run(p, stream=stream, sync=True)
        torch.cuda.synchronize()
        assert equal(got, want)
    with torch.cuda.stream(s):
        got = run(p)
    s.synchronize()
    assert equal(got, want)


def test_a_workspace_of_the_caller():
    p = problem(2)
    want = run(p)
    ws = torch.empty(mx.act8_wgrad_workspace(torch.bfloat16, 3000, 70, 130) + 64, dtype=torch.uint8, device="cuda")
    dw, db = torch.empty(70, 130, device="cuda"), torch.empty(70, device="cuda")
    mx.cu_fn_act8_wgrad_e(dw, p["dy"], p["c"], p["s"], DB=db, workspace=ws)
    assert equal((dw, db), want[:2])


def test_two_threads_at_once():
    ps = [problem(10), problem(20)]
    wants = [run(p, sync=True) for p in ps]
    results = [[], []]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                results[i].append(run(ps[i]))
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(len(r) == 20 for r in results)
    assert all(equal(got, wants[i]) for i in range(2) for got in results[i])


def test_captured_calls_replayed_with_other_inputs():
    """Two graphs with workspaces of their own, replayed in turn with eager calls between."""
    ps, graphs, outs = [problem(30), problem(40)], [], []
    for p in ps:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(p)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(p))
        graphs.append(g)
    for seed in range(50, 80, 10):
        for i, p in enumerate(ps):
            for key, t in problem(seed + i).items():
                p[key].copy_(t)
        wants = [run(p) for p in ps]
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert equal(outs[0], wants[0]) and equal(outs[1], wants[1])
        assert equal(run(ps[0]), wants[0])


@pytest.mark.parametrize("mx4", [False, True], ids=["act8", "mx4"])
def test_a_captured_training_step(mx4):
    params = leaves(torch.bfloat16)
    x, dy = values(1, 150, 100, torch.bfloat16, 0.1), values(2, 150, 60, torch.bfloat16, 0.1)

    def step():
        return torch.autograd.grad(mlp(x, *params, mx4), params, dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (5, 6, 7):
        x.copy_(values(seed, 150, 100, torch.bfloat16, 0.1))
        g.replay()
        torch.cuda.synchronize()
        assert equal(got, step())


@pytest.mark.parametrize("layer", [ptmx.act8_linear, ptmx.mx4_linear])
@pytest.mark.parametrize("shape", [(0, 48), (3, 0, 48), (1, 48), (48,)], ids=str)
def test_no_tokens_and_one_token(layer, shape):
    x = torch.randn(shape, device="cuda").requires_grad_()
    w = torch.randn(20, 48, device="cuda").requires_grad_()
    b = torch.randn(20, device="cuda").requires_grad_()
    y = layer(ptmx.act8_act(x, "silu"), w, b)
    assert y.shape == shape[:-1] + (20,)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == x.shape and dw.shape == w.shape
    tokens = x.numel() // 48
    assert torch.equal(db, torch.full_like(db, tokens))
    assert tokens or not dw.any()
    assert ptmx.Mx4Weight(w).linear(x.detach()).shape == y.shape


def test_second_derivatives_are_refused():
    x = torch.randn(4, 48, device="cuda").requires_grad_()
    dx, = torch.autograd.grad(ptmx.act8_act(x, "gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
