"""The fp8 block-128 operators: plain forms, cases and work counts.

A block-128 tensor is a pair (q, scales): q holds e4m3 values [rows, cols], scales one fp32 factor for each
128 consecutive values of a row, [rows, ceil(cols / 128)]; the pair stands for q * scale.

Operators (key "op" of a case):
  checkpoint   x -> (q, scales) with power-of-two scales, and back: what an 8-bit activation checkpoint keeps
  linear       y = x^ W^T (+ bias): x is quantised within the call, W is block-128 with the amax / 448 scales that
               weights restored or pushed as fp8 have
  input_grad   dx = dy W
  weight_grad  dw = dy^T x^, x^ an 8-bit checkpoint
  swiglu       h = silu(gate) * up keeping gate and up in 8 bits, and the gradients from what was kept
"""

import math

import torch

own = False

_BF16, _FP16, _FP32 = "bf16", "fp16", "fp32"
_DTYPE = {_BF16: torch.bfloat16, _FP16: torch.float16, _FP32: torch.float32}


def listed():
    return [
        # one token through an attention output projection of Qwen2.5-32B: latency, weight bytes
        dict(name="linear one token", op="linear", m=1, k=5120, n=5120, dtype=_BF16, bias=False),
        # a decode batch through a Llama-3-8B gate projection: weight bytes
        dict(name="linear decode batch", op="linear", m=64, k=4096, n=14336, dtype=_BF16, bias=False),
        # a chunk of a prompt through an eighth of a down projection, an odd number of tokens and of outputs
        dict(name="linear ragged", op="linear", m=1531, k=3456, n=5001, dtype=_FP16, bias=True),
        # a prompt of 4096 tokens through a whole Qwen2.5-32B up projection: tensor-core rate
        dict(name="linear prompt", op="linear", m=4096, k=5120, n=27648, dtype=_BF16, bias=False),
        # the gradient that a Llama-3-8B gate projection hands down for 4096 tokens
        dict(name="input_grad", op="input_grad", m=4096, n=14336, k=4096, dtype=_BF16),
        # the same of a small layer whose width is no multiple of 128
        dict(name="input_grad ragged", op="input_grad", m=77, n=520, k=1000, dtype=_BF16),
        # gradient of a down projection from 8192 checkpointed tokens, into fp32 for the optimizer
        dict(name="weight_grad", op="weight_grad", m=8192, n=4096, k=14336, dtype=_FP32),
        # few tokens, a small layer, an odd number of inputs
        dict(name="weight_grad ragged", op="weight_grad", m=333, n=520, k=1001, dtype=_BF16),
        # the gated activation of Llama-3-8B over 8192 tokens, forward and backward
        dict(name="swiglu", op="swiglu", m=8192, k=14336, dtype=_BF16),
        # the same for three tokens of an eighth of Qwen2.5-32B: latency
        dict(name="swiglu few tokens", op="swiglu", m=3, k=3456, dtype=_BF16),
        # the residual stream of 16384 tokens saved and loaded
        dict(name="checkpoint", op="checkpoint", m=16384, k=5120, dtype=_BF16),
        # a small odd fp32 activation
        dict(name="checkpoint ragged", op="checkpoint", m=5, k=1001, dtype=_FP32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "input_grad", "weight_grad", "swiglu", "checkpoint"])
    most = 4096 * 5120 * 27648  # multiply-adds of the largest listed product
    while True:
        m = _log(rng, 1, 8192)
        if op == "linear":
            k = 128 * _log(rng, 1, 216)
            n = _log(rng, 1, 27648)
            c = dict(op=op, m=m, k=k, n=n, dtype=rng.choice([_BF16, _BF16, _FP16]), bias=rng.random() < 0.5)
        elif op == "input_grad":
            k, n = _log(rng, 16, 14336), 8 * _log(rng, 1, 1792) + rng.choice([0, 0, 0, 3])
            c = dict(op=op, m=m, n=n, k=k, dtype=_BF16)
        elif op == "weight_grad":
            k, n = _log(rng, 16, 14336), 8 * _log(rng, 1, 1792) + rng.choice([0, 0, 0, 5])
            c = dict(op=op, m=m, n=n, k=k, dtype=rng.choice([_BF16, _FP32]))
        else:
            n = 1
            c = dict(op=op, m=m, k=_log(rng, 1, 14336), dtype=rng.choice([_BF16, _BF16, _FP16, _FP32]))
        if c["m"] * c["k"] * n <= most:
            return c


def work(case):
    m, k, n = case["m"], case["k"], case.get("n", 0)
    e = 4 if case["dtype"] == _FP32 else 2
    scales = 4 * -(-k // 128)
    op = case["op"]
    if op == "linear":
        return {"bytes": m * k * e + n * (k + scales) + m * n * e + (n * e if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "input_grad":
        return {"bytes": 2 * m * n + n * (k + scales) + 2 * m * k, "flops": 2 * m * n * k}
    if op == "weight_grad":
        return {"bytes": 2 * m * n + m * (k + scales) + e * n * k, "flops": 2 * m * n * k}
    if op == "swiglu":  # forward reads two, writes one and the 8-bit pair; backward reads one and the pair, writes two
        return {"bytes": m * (6 * k * e + 4 * (k + scales)), "flops": 30 * m * k}
    return {"bytes": m * (2 * k * e + 2 * (k + scales)), "flops": 4 * m * k}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, m, k, dtype):
    """N(0, 1) with a few outlier features and, where there are rows enough, some all-zero (padding) rows."""
    x = torch.randn(m, k, generator=g, device="cuda")
    x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 12.0, 1.0)
    if m > 8:
        x *= (torch.rand(m, 1, generator=g, device="cuda") >= 0.03)
    return x.to(dtype)


def _pitched(q):
    """Rows of q start on 16-byte boundaries, as the operators lay them out."""
    m, k = q.shape
    buf = torch.zeros(m, -(-k // 16) * 16, dtype=torch.uint8, device=q.device)
    buf[:, :k] = q.view(torch.uint8)
    return buf.view(torch.float8_e4m3fn)[:, :k]


def _blocks(x):
    """fp32 [m, blocks, 128] of x, zeros past the end of a row."""
    m, k = x.shape
    b = -(-k // 128)
    out = torch.zeros(m, b * 128, dtype=torch.float32, device=x.device)
    out[:, :k] = x
    return out.view(m, b, 128)


def _weight(g, n, k):
    """A bf16 weight as fp8 with scale amax / 448, the form in which the framework restores and pushes weights."""
    w = _blocks((torch.randn(n, k, generator=g, device="cuda") * 0.02).to(torch.bfloat16))
    amax = w.abs().amax(dim=2)
    scale = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    q = (w / scale[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return _pitched(q.view(n, -1)[:, :k]), scale


def _quantize(x):
    """Plain form: power-of-two scale, the smallest for which the block's amax is within 448."""
    b = _blocks(x)
    amax = b.abs().amax(dim=2)
    f, e = torch.frexp(amax)  # amax = f 2^e, 448 = 0.875 2^9
    e = torch.where(f > 0.875, e - 8, e - 9).clamp(min=-117)
    scale = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.ones_like(amax))
    q = (b / scale[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(x.shape[0], -1)[:, :x.shape[1]], scale


def _dequantize(q, scale):
    """Plain form: the fp32 values that (q, scale) stands for."""
    return (_blocks(q.float()) * scale[:, :, None]).view(q.shape[0], -1)[:, :q.shape[1]]


def prepare(case, seed):
    g = _generator(seed)
    m, k, op, dtype = case["m"], case["k"], case["op"], _DTYPE[case["dtype"]]
    s = {"op": op, "dtype": dtype}
    if op == "linear":
        s["x"] = _activations(g, m, k, dtype)
        s["q"], s["scale"] = _weight(g, case["n"], k)
        s["bias"] = (torch.randn(case["n"], generator=g, device="cuda") * 0.1).to(dtype) if case["bias"] else None
    elif op == "input_grad":
        s["dy"] = _activations(g, m, case["n"], torch.bfloat16) * 1e-2
        s["q"], s["scale"] = _weight(g, case["n"], k)
    elif op == "weight_grad":
        s["dy"] = _activations(g, m, case["n"], torch.bfloat16) * 1e-2
        q, s["scale"] = _quantize(_activations(g, m, k, torch.bfloat16))
        s["q"] = _pitched(q)
    elif op == "swiglu":
        s["gate"] = _activations(g, m, k, dtype)
        s["up"] = _activations(g, m, k, dtype)
        s["dh"] = _activations(g, m, k, dtype) * 1e-2
    else:
        s["x"] = _activations(g, m, k, dtype)
    return s


def _run_own(s):
    from statespectre_b200 import ops

    op = s["op"]
    if op == "linear":
        return ops.linear(s["x"], (s["q"], s["scale"]), s["bias"])
    if op == "input_grad":
        return ops.linear_input_grad(s["dy"], (s["q"], s["scale"]))
    if op == "weight_grad":
        return ops.linear_weight_grad(s["dy"], (s["q"], s["scale"]), out_dtype=s["dtype"])
    if op == "swiglu":
        h, kept = ops.swiglu_forward(s["gate"], s["up"])
        dgate, dup = ops.swiglu_backward(s["dh"], kept)
        return {"h": h, "dgate": dgate, "dup": dup}
    q, scale = ops.quantize(s["x"])
    return {"values": ops.dequantize((q, scale), s["dtype"]), "scale": scale}


def run(s):
    if own:
        return _run_own(s)
    op, dtype = s["op"], s["dtype"]
    if op == "linear":
        y = _dequantize(*_quantize(s["x"])) @ _dequantize(s["q"], s["scale"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(dtype)
    if op == "input_grad":
        return (s["dy"].float() @ _dequantize(s["q"], s["scale"])).to(dtype)
    if op == "weight_grad":
        return (s["dy"].float().t() @ _dequantize(s["q"], s["scale"])).to(dtype)
    if op == "swiglu":
        gate, up, dh = s["gate"].float(), s["up"].float(), s["dh"].float()
        h = gate / (1 + torch.exp(-gate)) * up
        gate, up = _dequantize(*_quantize(gate)), _dequantize(*_quantize(up))
        sig = 1 / (1 + torch.exp(-gate))
        dgate, dup = dh * up * sig * (1 + gate * (1 - sig)), dh * gate * sig
        return {"h": h.to(dtype), "dgate": dgate.to(dtype), "dup": dup.to(dtype)}
    q, scale = _quantize(s["x"])
    return {"values": _dequantize(q, scale).to(dtype), "scale": scale}


def _exact_values(q, scale):
    """64-bit values of a block-128 pair."""
    cols = torch.arange(q.shape[1], device=q.device) // 128
    return q.double() * scale.double()[:, cols]


def _exact_quantize(x):
    """64-bit values and scales of the power-of-two quantisation: e4m3 has three fraction bits, exponents down to
    2^-6 and values of 2^-9 below, and rounds to the nearest, ties to the even one."""
    x = x.double()
    m, k = x.shape
    group = (torch.arange(k, device=x.device) // 128).expand(m, k)
    amax = torch.zeros(m, -(-k // 128), dtype=torch.float64, device=x.device)
    amax.scatter_reduce_(1, group, x.abs(), "amax")
    e = torch.full_like(amax, -117)
    for step in (128, 64, 32, 16, 8, 4, 2, 1, 1):  # the smallest e >= -117 with amax <= 448 2^e
        e = torch.where(amax > 448 * torch.exp2(e + step - 1), e + step, e)
    scale = torch.where(amax > 0, torch.exp2(e), torch.ones_like(e))
    s = scale.gather(1, group)
    v = x / s
    _, ve = torch.frexp(v)
    unit = torch.exp2((ve - 1).clamp(min=-6).double() - 3)
    return torch.round(v / unit) * unit * s, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "linear":
        y = _exact_quantize(s["x"])[0] @ _exact_values(s["q"], s["scale"]).t()
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "input_grad":
        return s["dy"].double() @ _exact_values(s["q"], s["scale"])
    if op == "weight_grad":
        return s["dy"].double().t() @ _exact_values(s["q"], s["scale"])
    if op == "swiglu":
        gate, up, dh = s["gate"].double(), s["up"].double(), s["dh"].double()
        h = gate * torch.sigmoid(gate) * up
        gate, up = _exact_quantize(gate)[0], _exact_quantize(up)[0]
        sig = torch.sigmoid(gate)
        return {"h": h, "dgate": dh * up * (sig + gate * sig * (1 - sig)), "dup": dh * gate * sig}
    values, scale = _exact_quantize(s["x"])
    return {"values": values, "scale": scale}
