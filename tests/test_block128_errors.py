"""A product whose bounded wait ran out: the word that its kernel sets is set here from the host."""

import pytest
import torch

from statespectre_b200 import ops
from statespectre_b200._native import native


def test_no_error_where_no_product_ran():
    native().block128_set_error(40, 7)
    assert ops.product_error(40) == 0 and ops.product_error(-1) == 0 and ops.product_error("cuda:41") == 0


@pytest.mark.gpu
def test_later_products_raise_until_the_error_is_cleared():
    x, w = torch.randn(20, 256, device="cuda").to(torch.bfloat16), ops.quantize(torch.randn(64, 256, device="cuda"))
    y, g = ops.linear(x, w), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = ops.linear(x, w)
    torch.cuda.synchronize()
    assert ops.product_error() == 0
    native().block128_set_error(torch.cuda.current_device(), 203)
    try:
        for call in (lambda: ops.linear(x, w), lambda: ops.linear_input_grad(y, w),
                     lambda: ops.linear_weight_grad(y, ops.quantize(x))):
            with pytest.raises(RuntimeError, match="code 203"):
                call()
        ops.dequantize(w)  # waits for nothing
        g.replay()
        torch.cuda.synchronize()
        assert ops.product_error() == 203 and ops.product_error(torch.device("cuda")) == 203
        assert ops.product_error(x.device, clear=True) == 203
    finally:
        native().block128_set_error(torch.cuda.current_device(), 0)
    assert ops.product_error() == 0
    assert torch.equal(ops.linear(x, w), y) and torch.equal(captured, y)
