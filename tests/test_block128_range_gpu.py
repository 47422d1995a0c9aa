"""The range of the fp8 block-128 product: results are finite wherever the formula is, however far out the operands'
scales lie, since 3.4e38 is the largest value on either side."""

import pytest
import torch

from statespectre_b200 import ops
from test_block128_gpu import BF16, FP32, amax_pair, check_product, quantize64, randn, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 20, 50, 100, 600])
@pytest.mark.parametrize("size", [1e30, 1e34, 1e37, 8e37])
def test_large_activations(m, size):
    """randn stays under 6, so that 8e37 reaches past the largest bfloat16 in no element that is not clipped here."""
    x = (randn((m, 640), 1, 1.0, FP32).clamp(-4, 4) * size).to(BF16)
    x[0, :128] = 3.3e38
    w = amax_pair(300, 640, 2, 1e-4 / 640)
    y = ops.linear(x, w, out_dtype=FP32)
    ref = quantize64(x)[0] @ values(w).t()
    assert bool((ref.abs() < 3e38).all()) and bool(y.isfinite().all())
    check_product(y, quantize64(x)[0], values(w).t(), FP32, 640)


@pytest.mark.parametrize("m", [1, 20, 50, 100, 600])
@pytest.mark.parametrize("shift", [-118, -110, -96, -60, 60, 96, 105])
def test_far_scales_that_meet(m, shift):
    """x times 2^shift, the weights times 2^-shift: the results of no shift, bit for bit, as long as nothing leaves
    e4m3's range (a block's scale is at least 2^-117, so x is taken 2^9 up where it goes that far)."""
    x = randn((m, 384), 1, 1.0, FP32)
    q, s = amax_pair(300, 384, 2, 1.0)
    want = ops.linear(x, (q, s), out_dtype=FP32)
    up = 2.0 ** (16 if shift < -100 else 0)  # keeps the far blocks' own scale over 2^-117
    big = ops.linear(x * up * 2.0 ** (shift / 2) * 2.0 ** (shift / 2), (q, s * 2.0 ** -shift / up), out_dtype=FP32)
    assert torch.equal(big, want)


@pytest.mark.parametrize("m", [1, 20, 50, 100, 600])
def test_far_scales_beside_near_ones(m):
    """A few rows of the weight whose scales times 2^16 would overflow, in some blocks that meet small activations, and
    others beside them that meet large ones."""
    x = randn((m, 384), 1, 2.0 ** -60, FP32)
    x[:, :128] = randn((m, 128), 2, 2.0 ** 115, FP32)
    x[0, :128] = 3e38
    q, s = amax_pair(300, 384, 2, 1.0)
    s[:, 0] *= 2.0 ** -30
    s[::7, 1] *= 2.0 ** 120
    s[5, 2] *= 2.0 ** 118
    y = ops.linear(x, (q, s), out_dtype=FP32)
    assert bool(y.isfinite().all())
    check_product(y, quantize64(x)[0], values((q, s)).t(), FP32, 384)
    x[:] = 0
    assert not ops.linear(x, (q, s), out_dtype=FP32).any()
