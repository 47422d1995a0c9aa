"""Sums of the block-128 products: every way in which the kernels cut one into parts, at sizes taken from the number of
SMs, so that each test reaches the way that it is meant for on any device.

Small integers with power-of-two scales have exact sums in fp32 as long as they stay below 2^24, whatever the order and
the rounding of the additions: those results have to be equal, which shows a missing or a doubled term and a partial sum
kept in too few bits at any length."""

import pytest
import torch

from statespectre_b200 import ops
from test_block128_gpu import BF16, FP16, FP32, check_product, gen, randn, values

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def up(a, b):
    return -(-a // b)


def integers(shape, seed, top=8):
    return torch.randint(-top, top + 1, shape, generator=gen(seed), device="cuda").to(BF16)


def grad_way(ni, nj, nt):
    """(CTAs on a tile, parts of the sum, steps of the longest part, tiles of a CTA or pair)."""
    tiles, steps = up(ni, 128) * up(nj, 128), up(nt, 64)
    if tiles * 2 > sms():
        return 2, 1, steps, up(up(ni, 256) * up(nj, 256), sms() // 2)
    split = max(1, min(8, sms() // tiles, steps // 8))
    return 1, split, up(steps, split), 1


def linear_way(m, n):
    """(tokens of a tile, rounds of tiles)."""
    for bn, per_sm in ((16, 2), (32, 2), (64, 1)):
        if m <= bn:
            return bn, up(up(n, 128), sms() * per_sm)
    pairs, tiles = up(m, 224) * up(n, 256), up(m, 128) * up(n, 128)
    r2, r1 = up(2 * pairs, sms()), up(tiles, sms())
    return (224, r2) if r2 * 11 < r1 * 9 else (128, r1)


def wide(tiles):
    """Columns of that many 128 x 128 tiles in two rows of tiles."""
    return up(tiles, 2) * 128


def both_gradients(ni, nj, nt, a, b, out):
    """The same sum through the two kernels: a [nt, ni] and the pair b [nt, nj]."""
    return ops.linear_weight_grad(a, b, out), ops.linear_input_grad(a.t().contiguous(), b, out)


@pytest.mark.parametrize("out", [BF16, FP16, FP32])
@pytest.mark.parametrize("nt", [8192, 8193, 16500])
def test_long_unsplit_sums(nt, out):
    """Pairs of CTAs, one part: runs of 8192 terms added up in tensor memory (16-bit results), of 2048 in the output."""
    ni, nj = 200, wide(sms() // 2 + 1)
    ctas, split, steps, _ = grad_way(ni, nj, nt)
    assert (ctas, split) == (2, 1) and steps >= 128
    a, b = randn((nt, ni), 1), ops.quantize(randn((nt, nj), 2))
    for got in both_gradients(ni, nj, nt, a, b, out):
        check_product(got, a.double().t(), values(b), out, nt)
        ref = a.double().t() @ values(b)
        limit = (ref.to(out).double() - ref).norm() if out != FP32 else 0.0
        # truncated additions: at most a unit of 2^-23 of a partial sum for each 16 terms of a run
        run = 2048 if out == FP32 else 8192
        assert (got.double() - ref).norm() <= 1.01 * limit + run / 16 * 2.0 ** -23 * ref.norm()


@pytest.mark.parametrize("nj_off", [0, 1])
def test_fp32_sums_are_taken_in_runs_of_2048(nj_off):
    """Terms with a mean, so that truncations add up. A run makes 128 additions, which lose half of at most 2^-23 of a
    partial sum on average, and a partial sum is half of its run's: 32 units of 2^-23. The runs are added to nearest,
    half a unit each; 8 units more are granted. Rows of the output that start on 16 bytes, and rows that do not; scales
    that are no powers of two, whose terms come in three parts each, in runs of 640."""
    for ni, nj, nt in ((200, wide(sms() // 2 + 1) + nj_off, 16500), (128, 300 + nj_off, 8 * 8192)):
        ctas, split, steps, _ = grad_way(ni, nj, nt)
        assert steps >= 100 and (split == 1) == (ctas == 2)
        a, b = randn((nt, ni), 1) + 1, ops.quantize(randn((nt, nj), 2) + 1)
        for scales, run in ((b[1], 2048), (b[1] * 1.37, 640)):
            ref = a.double().t() @ values((b[0], scales))
            for got in both_gradients(ni, nj, nt, a, (b[0], scales), FP32):
                assert float(((got.double() - ref) / ref).abs().mean()) <= (32 + nt / run / 2 + 8) * 2.0 ** -23


@pytest.mark.parametrize("out", [BF16, FP32])
def test_several_tiles_with_sums_of_many_steps(out):
    """A pair walks several tiles: rings and buffers of tensor memory go on from one tile to the next."""
    ni, nj, nt = 1100, 256 * (sms() // 4), 777
    ctas, _, steps, tiles = grad_way(ni, nj, nt)
    assert ctas == 2 and steps >= 10 and tiles >= 2
    a, b = randn((nt, ni), 1), ops.quantize(randn((nt, nj), 2))
    for got in both_gradients(ni, nj, nt, a, b, out):
        check_product(got, a.double().t(), values(b), out, nt)


# outputs of one tile to several rounds of pairs, sums of one step to many, widths that are no multiples of anything
INT_SHAPES = [(1, 1, 1), (130, 257, 70), (128, 300, 14336), (77, 1001, 5121), (40, 2000, 9001), (300, 2600, 4160),
              (1100, 2300, 4161), (2050, 4701, 333)]


@pytest.mark.parametrize("ni,nj,nt", INT_SHAPES)
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
def test_integer_gradients_are_exact(ni, nj, nt, out):
    top = 8 if nt * 64 < 2 ** 24 else 2
    a, b = integers((nt, ni), 1, top), ops.quantize(integers((nt, nj), 2, top))
    ref = a.double().t() @ values(b)
    assert float(ref.abs().max()) < 2 ** 24 and float((a.double().t().abs() @ values(b).abs()).max()) < 2 ** 24
    for got in both_gradients(ni, nj, nt, a, b, out):
        assert torch.equal(got, ref.to(out))


def linear_shapes():
    s = sms()
    return [(1, 640, 5120), (1, s * 256 + 5, 1024), (16, 14336, 512), (20, 1024, 14336), (33, 900, 1000), (64, 2000, 4096),
            (64, 260, 14336), (100, 200, 9000), (128, 257, 13824), (300, 520, 5120), (1024, 4096, 512),
            (1100, 128 * s, 700), (2100, 3333, 384), (900, 256 * (s // 4) + 9, 1152)]


@pytest.mark.parametrize("case", range(14))
@pytest.mark.parametrize("bias", [False, True])
def test_integer_products_are_exact(case, bias):
    m, n, k = linear_shapes()[case]
    x, w = integers((m, k), 1), ops.quantize(integers((n, k), 2))
    b = integers((n,), 3).float() if bias else None
    ref = x.double() @ values(w).t() + (b.double() if bias else 0)
    assert float((x.double().abs() @ values(w).abs().t()).max()) + 8 < 2 ** 24
    assert torch.equal(ops.linear(x, w, b, out_dtype=FP32), ref.float())
    y = ops.linear(x, w, None if b is None else b.to(BF16))
    assert torch.equal(y, ref.to(BF16))


def test_integer_products_take_every_form():
    ways = {linear_way(m, n) for m, n, _ in linear_shapes()}
    assert {bn for bn, _ in ways} == {16, 32, 64, 128, 224}
    assert any(bn == 128 and r > 1 for bn, r in ways) and any(bn == 224 and r > 1 for bn, r in ways)
    assert any(bn == 16 and r > 1 for bn, r in ways)
    ways = {grad_way(*s) for s in INT_SHAPES}
    assert {w[0] for w in ways} == {1, 2} and max(w[1] for w in ways) == 8 and max(w[3] for w in ways) > 1
    assert any(w[0] == 1 and w[1] == 1 for w in ways) and any(w[0] == 2 and w[2] > 60 for w in ways)


@pytest.mark.parametrize("m,n,k", [(1, 512, 5120), (24, 300, 14336), (64, 1000, 4096), (100, 300, 5120),
                                   (300, 900, 1792), (1024, 4096, 512)])
def test_the_error_of_a_product(m, n, k):
    """In fp32, as a whole: a 128-block is eight additions that truncate in the tensor core (four steps, and the scale of
    each), at most a unit of 2^-23 of the block's partial sums; blocks are added to nearest, half a unit of the partial
    sum each. Blocks are independent, so all of it grows like the square root of the blocks times their size, as the
    result does: 8 + sqrt(blocks) / 2 units of the result."""
    x, w = randn((m, k), 1), ops.quantize(randn((n, k), 2))
    w = (w[0], w[1] * 1.37)
    xq = ops.quantize(x)
    ref = values(xq) @ values(w).t()
    got = ops.linear(x, w, out_dtype=FP32).double()
    assert (got - ref).norm() <= (8 + up(k, 128) ** 0.5 / 2) * 2.0 ** -23 * ref.norm()
