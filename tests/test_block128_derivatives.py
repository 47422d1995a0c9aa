"""Derivatives that the operators do not have are refused, not lost: forward mode, and gradients of a pair."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from statespectre_b200 import ops
from statespectre_b200.ops import block128

FP8 = torch.float8_e4m3fn


def x(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def pair(rows, cols):
    return torch.zeros(rows, cols, dtype=FP8), torch.ones(rows, -(-cols // 128))


def dual(t):
    return fw.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("call", [
    lambda: ops.linear(dual(x(2, 128)), pair(4, 128)), lambda: ops.linear(x(2, 128), dual(x(4, 128))),
    lambda: ops.linear(x(2, 128), pair(4, 128), dual(x(4))), lambda: ops.quantize(dual(x(2, 128))),
    lambda: ops.linear(x(2, 128), (pair(4, 128)[0], dual(torch.ones(4, 1)))),
    lambda: ops.dequantize((pair(4, 128)[0], dual(torch.ones(4, 1)))), lambda: ops.swiglu(dual(x(2, 8)), x(2, 8)),
    lambda: ops.swiglu(x(2, 8), dual(x(2, 8))), lambda: ops.swiglu_forward(x(2, 8), dual(x(2, 8))),
    lambda: ops.swiglu_backward(dual(x(2, 8)), (pair(2, 8), pair(2, 8))),
    lambda: ops.linear_input_grad(dual(x(2, 4)), pair(4, 128)), lambda: ops.linear_weight_grad(dual(x(2, 4)), pair(2, 8))])
def test_forward_mode_is_refused(monkeypatch, call):
    real = block128._on_gpu

    def any_device(t, what):
        try:
            return real(t, what)
        except ValueError as e:
            if "CUDA" in str(e):
                return t
            raise

    monkeypatch.setattr(block128, "_on_gpu", any_device)
    monkeypatch.setattr(block128, "_launch", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(block128, "_launch_grad", lambda *a: pytest.fail("launched"))
    with fw.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            call()


def test_tensors_without_a_tangent_pass_inside_a_dual_level():
    with fw.dual_level():
        with pytest.raises(ValueError, match="CUDA tensor"):
            ops.quantize(x(2, 128))
        with pytest.raises(ValueError, match="CUDA tensor"):
            ops.dequantize(pair(2, 128))


@pytest.mark.parametrize("call", [
    lambda p: ops.linear(x(2, 128), p), lambda p: ops.dequantize(p), lambda p: ops.linear(x(2, 128).requires_grad_(), p)])
def test_gradients_of_a_pair_are_refused(monkeypatch, call):
    monkeypatch.setattr(block128, "_on_gpu", lambda t, what: t)
    q, s = pair(4, 128)
    with pytest.raises(ValueError, match="gradient"):
        call((q, s.requires_grad_()))


def test_a_pair_that_requires_gradients_serves_without_them(monkeypatch):
    monkeypatch.setattr(block128, "_on_gpu", lambda t, what: t)
    q, s = pair(4, 128)
    with torch.no_grad():
        assert block128._pair((q, s.requires_grad_()), "x")[2:4] == (4, 128)


@pytest.mark.gpu
def test_forward_mode_on_the_gpu():
    a, w = torch.randn(3, 128, device="cuda").to(torch.bfloat16), torch.randn(8, 128, device="cuda").to(torch.bfloat16)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda t: ops.linear(t, w), (a,), (torch.ones_like(a),))
    with fw.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            ops.swiglu(dual(a), a)
        y = ops.linear(a, w)
    assert torch.equal(y, ops.linear(a, w))
