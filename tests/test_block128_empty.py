"""Rows without columns are rows: an empty layer trains like any other."""

import pytest
import torch

from statespectre_b200 import ops
from statespectre_b200.ops import block128


@pytest.mark.parametrize("shape", [(2, 3, 0), (6, 0), (0, 0), (0,), (1, 0), (2, 0, 0)])
def test_rows_without_columns_are_counted(shape):
    _, rows, cols, _ = block128._matrix(torch.zeros(shape), "x")
    assert cols == 0 and rows == torch.Size(shape[:-1]).numel()


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(2, 3), (6,), (), (0,), (2, 0)])
@pytest.mark.parametrize("n,k", [(0, 5), (4, 0), (0, 0), (4, 5)])
def test_empty_layers_train(lead, n, k):
    def leaf(*shape):
        return torch.randn(*shape, device="cuda").to(torch.bfloat16).requires_grad_()

    x, w, b = leaf(*lead, k), leaf(n, k), leaf(n)
    y = ops.linear(x, w, b)
    assert y.shape == (*lead, n)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape and torch.equal(db, torch.full_like(b, y.numel() // n if n else 0))
    if not n:
        assert not dx.any()
    g = leaf(*lead, k)
    dg, = torch.autograd.grad(ops.swiglu(g, x), g, torch.ones_like(g))
    assert dg.shape == g.shape
