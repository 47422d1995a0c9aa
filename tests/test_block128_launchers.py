"""Pitches that do not fit 32 bits, and negative ones, are refused by every elementwise launcher before anything runs."""

import pytest

from statespectre_b200._native import native

A = 1 << 20  # an aligned address that no refused launch touches
BAD = [-256, (1 << 32) + 256, 1 << 32, -(1 << 32) + 256, 255]


def dequantize(q, x, **_):
    native().k_dequantize_block128(A, q, A, A, x, 0, 4, 256, 0)


def quantize(q, x, **_):
    native().k_quantize_block128(A, x, 0, A, q, A, 4, 256, 0)


def forward(q, x, y=256, h=256, **_):
    native().k_swiglu_forward(A, x, A, y, 0, A, h, A, A, A, A, q, 4, 256, 0)


def backward(q, x, u=256, d=256):
    native().k_swiglu_backward(A, x, 0, A, q, A, A, u, A, A, A, d, 4, 256, 0)


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("call,args", [(dequantize, ("q", "x")), (quantize, ("q", "x")), (forward, ("q", "x", "y", "h")),
                                       (backward, ("q", "x", "u", "d"))])
def test_pitches_are_refused(call, args, bad):
    for name in args:
        with pytest.raises(RuntimeError, match="invalid argument"):
            call(**(dict(q=256, x=256) | {name: bad}))


@pytest.mark.parametrize("bad", [b for b in BAD if b < 256] + [1 << 41, 1 << 62])
@pytest.mark.parametrize("name", ["x", "q", "w", "y"])
def test_product_pitches_are_refused(name, bad):
    if name == "y" and bad > 256:
        return  # a result may have any pitch
    p = dict(x=256, q=256, w=256, y=256) | {name: bad}
    C = native()
    with pytest.raises(RuntimeError, match="invalid argument"):
        C.k_linear_block128(A, p["x"], 0, A, p["q"], A, A, 1 << 20, A, p["w"], A, 0, A, p["y"], 0, 4, 256, 256, 0)
    if name in ("x", "w", "y"):
        with pytest.raises(RuntimeError, match="invalid argument"):
            C.k_matmul_input_grad(A, p["x"], A, p["w"], A, A, p["y"], 0, 4, 256, 256, 0)
        with pytest.raises(RuntimeError, match="invalid argument"):
            C.k_matmul_weight_grad(A, p["x"], A, p["w"], A, A, p["y"], 0, 4, 256, 256, 0)


def test_words_of_a_gradient_are_whole():
    for fn in (native().k_matmul_input_grad, native().k_matmul_weight_grad):
        with pytest.raises(RuntimeError, match="invalid argument"):
            fn(A, 256, A, 256, A, A, 256, 0, 4, 256, 256, 0, work=A + 2, words=148)
