"""Refusals of the block-128 operators (no GPU): Python's checks of types and shapes, the launchers' checks of
pointers, pitches and sizes."""

import pytest
import torch

from statespectre_b200 import ops
from statespectre_b200._native import native
from statespectre_b200.ops import block128

FP8 = torch.float8_e4m3fn


def pair(rows, cols):
    return torch.zeros(rows, cols, dtype=FP8), torch.ones(rows, -(-cols // 128))


def x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: ops.quantize(x(2, 128)), lambda: ops.dequantize(pair(2, 128)), lambda: ops.linear(x(2, 128), pair(4, 128)),
    lambda: ops.linear_input_grad(x(2, 4), pair(4, 128)), lambda: ops.linear_weight_grad(x(2, 4), pair(2, 128)),
    lambda: ops.swiglu(x(2, 8), x(2, 8)), lambda: ops.swiglu_backward(x(2, 8), (pair(2, 8), pair(2, 8)))])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="CUDA tensor"):
        call()


@pytest.mark.parametrize("call,error,text", [
    (lambda: ops.quantize([1.0]), TypeError, "must be a tensor"),
    (lambda: ops.quantize(x(2, 128, dtype=torch.float64)), ValueError, "bfloat16, float16 or float32"),
    (lambda: ops.quantize(x(2, 128, dtype=torch.int32)), ValueError, "bfloat16, float16 or float32"),
    (lambda: ops.quantize(torch.tensor(1.0)), ValueError, "one dimension"),
    (lambda: ops.dequantize(x(2, 128)), TypeError, "pair"),
    (lambda: ops.dequantize((x(2, 128), torch.ones(2, 1))), ValueError, "float8_e4m3fn"),
    (lambda: ops.dequantize((pair(2, 128)[0], torch.ones(2, 1).half())), ValueError, "float32"),
    (lambda: ops.dequantize((pair(2, 129)[0], torch.ones(2, 1))), ValueError, "do not fit"),
    (lambda: ops.dequantize(pair(2, 128), torch.int8), ValueError, "bfloat16, float16 or float32"),
    (lambda: ops.linear(x(2, 128), pair(4, 256)), ValueError, "256 columns"),
    (lambda: ops.linear(x(2, 128), (x(3, 4, 128).to(FP8), torch.ones(12, 1))), ValueError, "two dimensions"),
    (lambda: ops.linear(x(2, 128), 7), TypeError, "pair"),
    (lambda: ops.linear(x(2, 128), pair(4, 128), out_dtype=torch.float64), ValueError, "out_dtype"),
    (lambda: ops.linear(x(2, 128, dtype=torch.float16).requires_grad_(), pair(4, 128)), ValueError, "gradients"),
    (lambda: ops.linear_input_grad(x(2, 4, dtype=torch.float32), pair(4, 128)), ValueError, "dy must be bfloat16"),
    (lambda: ops.linear_input_grad(x(2, 5), pair(4, 128)), ValueError, "dy has 5 columns"),
    (lambda: ops.linear_weight_grad(x(2, 4), pair(3, 128)), ValueError, "dy has 2 rows"),
    (lambda: ops.linear_weight_grad(x(2, 4), pair(2, 128), torch.int8), ValueError, "out_dtype"),
    (lambda: ops.swiglu(x(2, 8), x(2, 9)), ValueError, "must match gate"),
    (lambda: ops.swiglu(x(2, 8), x(2, 8, dtype=torch.float32)), ValueError, "must match gate"),
    (lambda: ops.swiglu_backward(x(2, 8), (pair(2, 8), pair(2, 9))), ValueError, "dh has shape"),
    (lambda: ops.swiglu_backward(x(3, 8), (pair(2, 8), pair(2, 8))), ValueError, "dh has shape"),
    (lambda: ops.swiglu_backward(x(2, 8), pair(2, 8)[0]), TypeError, "two pairs"),
])
def test_arguments_are_refused(monkeypatch, call, error, text):
    """Types and shapes are checked before anything is launched."""
    real = block128._on_gpu

    def any_device(t, what):
        return t if isinstance(t, torch.Tensor) else real(t, what)

    monkeypatch.setattr(block128, "_on_gpu", any_device)
    monkeypatch.setattr(block128, "quantize", lambda t: pair(t.numel() // t.shape[-1], t.shape[-1])
                        if t.dtype in block128._TYPE and t.dim() else ops.quantize(t))
    with pytest.raises(error, match=text):
        call()


A = 1 << 20  # an aligned address that no refused launch touches


@pytest.mark.parametrize("args", [
    dict(x=0), dict(q=0), dict(s=0), dict(q=A + 8), dict(ldq=200), dict(ldx=255), dict(ldq=240), dict(rows=-1),
    dict(cols=-1), dict(rows=1 << 40), dict(kind=7)])
def test_quantize_launcher_refuses(args):
    a = dict(x=A, ldx=256, kind=0, q=A, ldq=256, s=A, rows=4, cols=256) | args
    for fn in ("quantize", "dequantize"):
        with pytest.raises(RuntimeError, match="invalid argument"):
            if fn == "quantize":
                native().k_quantize_block128(a["x"], a["ldx"], a["kind"], a["q"], a["ldq"], a["s"], a["rows"],
                                             a["cols"], 0)
            else:
                native().k_dequantize_block128(a["q"], a["ldq"], a["s"], a["x"], a["ldx"], a["kind"], a["rows"],
                                               a["cols"], 0)


@pytest.mark.parametrize("args", [
    dict(a=0), dict(q=0), dict(s=0), dict(o=0), dict(q=A + 4), dict(ldq=200), dict(lda=255), dict(ldo=1),
    dict(m=-1), dict(n=1 << 40), dict(red=0), dict(w=0), dict(w=A + 8), dict(wb=100)])
def test_product_launchers_refuse(args):
    a = dict(a=A, lda=256, q=A, ldq=256, s=A, o=A, ldo=256, m=256, n=256, red=256, w=A, wb=1 << 20) | args
    C = native()
    red = a["red"]
    with pytest.raises(RuntimeError, match="invalid argument"):  # red: the length that is summed over
        C.k_linear_block128(a["a"], a["lda"], 0, a["a"], a["lda"], a["s"], a["w"], a["wb"], a["q"], a["ldq"], a["s"], 0,
                            a["o"], a["ldo"], 0, a["m"], a["n"], red, 0)
    if "w" in args or "wb" in args:
        return
    with pytest.raises(RuntimeError, match="invalid argument"):
        C.k_matmul_input_grad(a["a"], a["lda"], a["q"], a["ldq"], a["s"], a["o"], a["ldo"], 0, a["m"], red, a["n"], 0)
    with pytest.raises(RuntimeError, match="invalid argument"):
        C.k_matmul_weight_grad(a["a"], a["lda"], a["q"], a["ldq"], a["s"], a["o"], a["ldo"], 0, red, a["m"], a["n"], 0)


def test_empty_shapes_launch_nothing():
    n = native().kernel_launch_count()
    native().k_quantize_block128(0, 128, 0, 0, 128, 0, 0, 128, 0)
    native().k_swiglu_forward(0, 8, 0, 8, 0, 0, 8, 0, 0, 0, 0, 16, 0, 8, 0)
    native().k_linear_block128(0, 128, 0, 0, 128, 0, 0, 0, 0, 128, 0, 0, 0, 4, 0, 0, 4, 128, 0)
    native().k_matmul_input_grad(0, 4, 0, 128, 0, 0, 128, 0, 0, 4, 128, 0)
    native().k_matmul_weight_grad(0, 4, 0, 128, 0, 0, 128, 0, 3, 0, 128, 0)
    assert native().kernel_launch_count() == n
