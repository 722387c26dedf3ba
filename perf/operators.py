"""Measured cases of the microscaled operators (necklace_amd.cuda.mx): 4-bit floating point
(quantise, decode, product) and 8-bit activation checkpoints (save, the activation's gradient and the
weight gradient that read them).

A matrix is cut along its rows into blocks of 32 neighbouring columns; a block has one power of two as
its scale, kept as a byte (the exponent plus 127; 255 says that the block held an infinity or a NaN).
4 bits: sign and 0, .5, 1, 1.5, 2, 3, 4, 6 times the scale 2^(floor(log2 max|x|) - 2), ties to even,
saturated at 6; two codes a byte, the even column in the low half.  8 bits: whole numbers -127 .. 127
times the scale 2^(floor(log2 max|x|) - 6).  Rows are padded with zeros to whole steps of 128 columns.

`own` False: the operators in elementary torch operations; True: the framework's calls.
"""
import math

import torch

own = False

BLOCK, STEP = 32, 128
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def _mx():
    from necklace_amd.cuda import mx  # only the framework's own calls need the package
    return mx


def listed():
    return [
        # a small layer's weight, as an optimizer step lays it out again: the latency of two short calls
        {"name": "mx4_small_weight", "op": "roundtrip", "dtype": "fp32", "rows": 33, "cols": 1000, "transpose": False},
        # activations of a long batch of tokens (the large square bench shape's width) on their way to a product
        {"name": "mx4_large_activations", "op": "roundtrip", "dtype": "bf16", "rows": 16384, "cols": 8192, "transpose": False},
        # a weight's transpose, for the gradient of a product's input; rows that start off every boundary
        {"name": "mx4_transposed_odd", "op": "roundtrip", "dtype": "fp32", "rows": 8191, "cols": 4097, "transpose": True},
        # one token through the 1024 -> 4096 projection of a GPT-2-medium-sized model
        {"name": "mx4_linear_one_token", "op": "linear", "dtype": "bf16", "m": 1, "n": 4096, "k": 1024, "bias": True},
        # a small batch of tokens through a wide layer: bound by the weight's bytes
        {"name": "mx4_linear_37_tokens", "op": "linear", "dtype": "fp16", "m": 37, "n": 8192, "k": 8192, "bias": False},
        # a ragged prompt through odd widths, in and out in fp32
        {"name": "mx4_linear_odd", "op": "linear", "dtype": "fp32", "m": 1001, "n": 1023, "k": 4097, "bias": True},
        # the product alone, both sides laid out before: the matrix cores' rate
        {"name": "mx4_matmul_8192", "op": "matmul", "dtype": "bf16", "m": 8192, "n": 8192, "k": 8192},
        # the activation of an MLP of 4096 hidden features over 16384 tokens: forward with its
        # checkpoint, and the gradient from the checkpoint
        {"name": "act8_gelu_16384x4096", "op": "act", "dtype": "bf16", "rows": 16384, "cols": 4096, "fn": "gelu"},
        # the same in fp32 with odd sizes
        {"name": "act8_silu_odd", "op": "act", "dtype": "fp32", "rows": 1001, "cols": 4097, "fn": "silu"},
        # weight and bias gradient of that MLP's first layer from the 8-bit checkpoint of its input
        {"name": "act8_wgrad_16384", "op": "wgrad", "dtype": "bf16", "t": 16384, "n": 4096, "k": 1024, "bias": True},
        # odd sizes with fp32 gradients, the type the gradient compressor takes
        {"name": "act8_wgrad_fp32_odd", "op": "wgrad", "dtype": "fp32", "t": 5001, "n": 1023, "k": 4097, "bias": False},
        # a small layer on a short batch: latency
        {"name": "act8_wgrad_small", "op": "wgrad", "dtype": "fp16", "t": 64, "n": 256, "k": 256, "bias": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["roundtrip", "linear", "matmul", "act", "wgrad"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "roundtrip":
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 16384), "cols": _log_int(rng, 1, 8192),
                "transpose": rng.random() < 0.5}
    if op == "linear":
        return {"op": op, "dtype": dtype, "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 32, 8192),
                "k": _log_int(rng, 32, 8192), "bias": rng.random() < 0.5}
    if op == "matmul":
        return {"op": op, "dtype": dtype, "m": _log_int(rng, 128, 8192), "n": _log_int(rng, 128, 8192),
                "k": _log_int(rng, 128, 8192)}
    if op == "act":
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 8192), "cols": _log_int(rng, 1, 8192),
                "fn": rng.choice(["gelu", "silu"])}
    return {"op": op, "dtype": dtype, "t": _log_int(rng, 1, 16384), "n": _log_int(rng, 16, 4096),
            "k": _log_int(rng, 16, 4096), "bias": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 17)


def _activations(gen, rows, cols, dtype):
    """Normal values, a few channels ten times as large, and some rows of padding (all zero)."""
    x = torch.randn(rows, cols, generator=gen, device="cuda")
    x *= 1 + 9 * (torch.rand(cols, generator=gen, device="cuda") < 0.01)
    if rows > 8:
        x *= (torch.rand(rows, 1, generator=gen, device="cuda") >= 0.02)
    return x.to(dtype)


def _gradients(gen, rows, cols, dtype):
    """Heavy-tailed and small, as an output's gradient is."""
    z = torch.randn(rows, cols, generator=gen, device="cuda")
    return (z * z.abs() * 1e-2).to(dtype)


def _padded(k):
    return -(-k // STEP) * STEP


def prepare(case, seed):
    gen, dtype, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    s = dict(case)
    if op == "roundtrip":
        s["x"] = _activations(gen, case["rows"], case["cols"], dtype)
    elif op == "linear":
        w = torch.randn(case["n"], case["k"], generator=gen, device="cuda") * 0.02
        s["cb"], s["sb"] = _mx4_codes(w)
        s["x"] = _activations(gen, case["m"], case["k"], dtype)
        s["bias"] = (torch.randn(case["n"], generator=gen, device="cuda") * 0.1).to(dtype) if case["bias"] else None
    elif op == "matmul":
        s["ca"], s["sa"] = _mx4_codes(_activations(gen, case["m"], case["k"], torch.float32))
        s["cb"], s["sb"] = _mx4_codes(torch.randn(case["n"], case["k"], generator=gen, device="cuda") * 0.02)
    elif op == "act":
        s["x"] = _activations(gen, case["rows"], case["cols"], dtype)
        s["dy"] = _gradients(gen, case["rows"], case["cols"], dtype)
    else:
        s["c"], s["s"] = _act8_codes(_activations(gen, case["t"], case["k"], dtype))
        s["dy"] = _gradients(gen, case["t"], case["n"], dtype)
    return s


# ------------------------------------------------------------------ the plain forms

def _blocks(x, bits):
    """x in fp32, padded, as [rows, blocks, 32], and the exponent of every block's scale."""
    x = x.float()
    x = torch.nn.functional.pad(x, (0, _padded(x.shape[1]) - x.shape[1]))
    x = x.view(x.shape[0], -1, BLOCK)
    top = x.abs().amax(2, keepdim=True)
    e = torch.frexp(top)[1] - 1 - (2 if bits == 4 else 6)
    e = torch.where(top > 0, e, -127).clamp(-127, 127)
    return x, e, torch.isfinite(top)


def _times_power(x, e):
    """x * 2^e in two exact factors: 2^127 and 2^-127 apart are not both normal numbers of 32 bits."""
    h = e // 2
    return x * torch.exp2(h.float()) * torch.exp2((e - h).float())


def _mx4_magnitudes(a):
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.round(a / step) * step).clamp(max=6)


def _mx4_values(x):
    """x as its 4-bit codes stand for it, in fp32."""
    b, e, ok = _blocks(x, 4)
    v = _times_power(b, -e)
    v = _times_power(torch.copysign(_mx4_magnitudes(v.abs()), v), e)
    return torch.where(ok, v, math.nan).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _mx4_codes(x):
    b, e, ok = _blocks(x, 4)
    v = torch.where(ok, _times_power(b, -e), 0.0)
    m = _mx4_magnitudes(v.abs())
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(x.shape[0], -1)
    scale = torch.where(ok, e + 127, 255).to(torch.uint8).squeeze(2)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), scale.contiguous()


def _mx4_decode(c, s):
    """Codes [rows, bytes] and scales as fp32 values, all padded columns."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=c.device)
    code = torch.stack((c & 15, c >> 4), 2).reshape(c.shape[0], -1, BLOCK)
    e = (s.int() - 127).unsqueeze(2)
    v = _times_power(table[code.int()], e)
    return torch.where(e == 128, math.nan, v).reshape(c.shape[0], -1)


def _act8_whole(x):
    b, e, ok = _blocks(x, 8)
    return torch.round(_times_power(b, -e)).clamp(-127, 127), e, ok


def _act8_values(x):
    q, e, ok = _act8_whole(x)
    return torch.where(ok, _times_power(q, e), math.nan).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _act8_codes(x):
    q, e, ok = _act8_whole(x)
    c = torch.where(ok, q, 0.0).to(torch.int8).reshape(x.shape[0], -1)
    return c.contiguous(), torch.where(ok, e + 127, 255).to(torch.uint8).squeeze(2).contiguous()


def _act8_decode(c, s):
    e = (s.int() - 127).unsqueeze(2)
    v = _times_power(c.view(c.shape[0], -1, BLOCK).float(), e)
    return torch.where(e == 128, math.nan, v).reshape(c.shape[0], -1)


def _act(x, fn):
    if fn == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x / (1 + torch.exp(-x))


def _act_slope(x, fn):
    if fn == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    g = 1 / (1 + torch.exp(-x))
    return g * (1 + x * (1 - g))


def _plain(s):
    op, dtype = s["op"], DTYPES[s["dtype"]]
    if op == "roundtrip":
        return _mx4_values(s["x"].t() if s["transpose"] else s["x"]).to(dtype)
    if op == "linear":
        y = _mx4_values(s["x"]) @ _mx4_decode(s["cb"], s["sb"])[:, :s["k"]].t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(dtype)
    if op == "matmul":
        return (_mx4_decode(s["ca"], s["sa"]) @ _mx4_decode(s["cb"], s["sb"]).t()).to(dtype)
    if op == "act":
        return {"y": _act(s["x"].float(), s["fn"]).to(dtype),
                "dx": (s["dy"].float() * _act_slope(_act8_values(s["x"]), s["fn"])).to(dtype)}
    dy = s["dy"].float()
    out = {"dw": dy.t() @ _act8_decode(s["c"], s["s"])[:, :s["k"]]}
    if s["bias"]:
        out["db"] = dy.sum(0)
    return out


# ------------------------------------------------------------------ the framework's calls

def _calls(s):
    mx, op, dtype = _mx(), s["op"], DTYPES[s["dtype"]]
    if op == "roundtrip":
        rows, cols = (s["cols"], s["rows"]) if s["transpose"] else (s["rows"], s["cols"])
        c, sc = mx.mx4_empty(rows, cols)
        mx.cu_fn_mx4_quantize_e(s["x"], c, sc, transpose=s["transpose"], sync=False)
        out = torch.empty(rows, cols, dtype=dtype, device="cuda")
        mx.cu_fn_mx4_dequantize_e(out, c, sc, sync=False)
        return out
    if op == "linear":
        y = torch.empty(s["m"], s["n"], dtype=dtype, device="cuda")
        mx.cu_fn_mx4_linear_e(y, s["x"], s["cb"], s["sb"], bias=s["bias"], sync=False)
        return y
    if op == "matmul":
        y = torch.empty(s["m"], s["n"], dtype=dtype, device="cuda")
        mx.cu_fn_mx4_matmul_e(y, s["ca"], s["sa"], s["cb"], s["sb"], sync=False)
        return y
    if op == "act":
        c, sc = mx.act8_empty(s["rows"], s["cols"])
        y, dx = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        mx.cu_fn_act8_save_e(s["x"], c, sc, Y=y, fn=s["fn"], sync=False)
        mx.cu_fn_act8_grad_e(dx, s["dy"], c, sc, fn=s["fn"], sync=False)
        return {"y": y, "dx": dx}
    dw = torch.empty(s["n"], s["k"], dtype=torch.float32, device="cuda")
    db = torch.empty(s["n"], dtype=torch.float32, device="cuda") if s["bias"] else None
    mx.cu_fn_act8_wgrad_e(dw, s["dy"], s["c"], s["s"], DB=db, sync=False)
    return {"dw": dw, "db": db} if s["bias"] else {"dw": dw}


def run(state):
    return _calls(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    b, op = SIZE[case["dtype"]], case["op"]
    if op == "roundtrip":  # the matrix in and out, its codes written and read
        n = case["rows"] * case["cols"]
        rows, cols = (case["cols"], case["rows"]) if case["transpose"] else (case["rows"], case["cols"])
        return {"bytes": 2 * b * n + 2 * rows * _padded(cols) * 17 // 32, "flops": 4 * n}
    if op in ("linear", "matmul"):
        m, n, k = case["m"], case["n"], case["k"]
        code = _padded(k) * 17 // 32
        x = m * k * b if op == "linear" else m * code
        return {"bytes": x + n * code + m * n * b + (n * b if case.get("bias") else 0), "flops": 2 * m * n * k}
    if op == "act":  # x in, y and codes out; dy and codes in, dx out
        n = case["rows"] * case["cols"]
        return {"bytes": 4 * b * n + 2 * case["rows"] * _padded(case["cols"]) * 33 // 32, "flops": 40 * n}
    t, n, k = case["t"], case["n"], case["k"]
    return {"bytes": t * n * b + t * _padded(k) * 33 // 32 + 4 * n * k + (4 * n if case["bias"] else 0),
            "flops": 2 * t * n * k + (t * n if case["bias"] else 0)}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_scaled(x, top_exponent):
    """Blocks of x in 64 bits, each divided by its scale, and the scale."""
    x = x.double()
    r, k = x.shape
    pad = torch.zeros(r, _padded(k), dtype=torch.float64, device=x.device)
    pad[:, :k] = x
    pad = pad.unflatten(1, (-1, BLOCK))
    top = pad.abs().max(-1, keepdim=True).values
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149))).clamp(min=-127 + top_exponent) - top_exponent
    scale = torch.pow(torch.full_like(e, 2.0), e)
    return pad / scale, scale


def _exact_mx4(x):
    v, scale = _exact_scaled(x, 2)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    border = (grid[1:] + grid[:-1]) / 2
    a = v.abs()
    low, high = torch.bucketize(a, border, right=False), torch.bucketize(a, border, right=True)
    at = torch.where(low % 2 == 0, low, high)  # on a border the two differ: the even code
    return (torch.sign(v) * grid[at] * scale).flatten(1)[:, :x.shape[1]]


def _exact_mx4_decode(c, s):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=c.device)
    both = torch.empty(c.shape[0], c.shape[1], 2, dtype=torch.float64, device=c.device)
    for half, code in enumerate((torch.remainder(c, 16).long(), torch.div(c, 16, rounding_mode="floor").long())):
        both[:, :, half] = grid[code % 8] * (1 - 2 * (code // 8)).double()
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=c.device), s.double() - 127)
    return both.flatten(1) * scale.repeat_interleave(BLOCK, 1)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "roundtrip":
        return _exact_mx4(s["x"].t().contiguous() if case["transpose"] else s["x"])
    if op == "linear":
        y = _exact_mx4(s["x"]).matmul(_exact_mx4_decode(s["cb"], s["sb"])[:, :case["k"]].t().contiguous())
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "matmul":
        return _exact_mx4_decode(s["ca"], s["sa"]).matmul(_exact_mx4_decode(s["cb"], s["sb"]).t().contiguous())
    if op == "act":
        x, dy = s["x"].double(), s["dy"].double()
        v, scale = _exact_scaled(s["x"], 6)
        saved = (torch.round(v).clamp(-127, 127) * scale).flatten(1)[:, :case["cols"]]
        normal = lambda u: torch.erfc(-u / math.sqrt(2.0)) / 2  # noqa: E731
        if case["fn"] == "gelu":
            slope = normal(saved) + saved * torch.exp(-saved.square() / 2) / math.sqrt(2 * math.pi)
            return {"y": x * normal(x), "dx": dy * slope}
        g = torch.sigmoid(saved)
        return {"y": x * torch.sigmoid(x), "dx": dy * (g + saved * g * torch.sigmoid(-saved))}
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), s["s"].double() - 127)
    x = (s["c"].double() * scale.repeat_interleave(BLOCK, 1))[:, :case["k"]].contiguous()
    dy = s["dy"].double()
    out = {"dw": dy.t().contiguous().matmul(x)}
    if case["bias"]:
        out["db"] = dy.sum(0)
    return out
