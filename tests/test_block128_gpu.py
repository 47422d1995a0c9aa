"""The block-128 operators against their formulas in 64 bits.

Tolerances. A rounding to type t is off by at most finfo(t).eps / 2 of the value. A sum of n products in fp32 whose
additions may truncate is off by at most (n + 4 ceil(n / 128) + 64) 2^-23 of the sum of the products' magnitudes: one
unit for each addition, four for applying each 128-block's scales, the rest for the last few operations. A weight
whose scale is no power of two is rounded to bfloat16 before it meets the gradient: 2^-8 of each product's magnitude.
"""

import math

import pytest
import torch

from statespectre_b200 import ops

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, seed=0, std=1.0, dtype=BF16):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def values(pair):
    """64-bit values of a pair."""
    q, s = pair
    cols = torch.arange(q.shape[-1], device=q.device) // 128
    return q.double() * s.double().reshape(*q.shape[:-1], -1)[..., cols]


def quantize64(x):
    """The quantisation's definition in 64 bits: (values, scales)."""
    x = x.double().reshape(-1, x.shape[-1])
    m, k = x.shape
    vals, scales = torch.empty_like(x), torch.ones(m, -(-k // 128), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        v = x[:, b * 128:(b + 1) * 128]
        amax = torch.where(v.isfinite(), v.abs(), 0).amax(1)
        e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 1) / 448)).clamp(min=-117)
        e = torch.where(amax > 448 * torch.exp2(e), e + 1, e)  # log2 is not exact next to a border
        e = torch.where((amax <= 448 * torch.exp2(e - 1)) & (e > -117), e - 1, e)
        s = torch.where(amax > 0, torch.exp2(e), torch.ones_like(e))
        u = v / s[:, None]
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
        step = torch.where(u.abs() >= step * 16, step * 2, torch.where(u.abs() < step * 8, step / 2, step))
        step = step.clamp(min=2.0 ** -9)
        vals[:, b * 128:(b + 1) * 128] = torch.where(v.isfinite(), torch.round(u / step) * step * s[:, None], math.nan)
        scales[:, b] = s
    return vals, scales


def amax_pair(n, k, seed, std=0.02):
    """A weight as the fp8 restore and push leave it: scale amax / 448."""
    w = randn((n, k), seed, std).float()
    pad = torch.zeros(n, -(-k // 128) * 128, device="cuda")
    pad[:, :k] = w
    b = pad.view(n, -1, 128)
    s = b.abs().amax(2) / 448
    s = torch.where(s > 0, s, 1)
    q = (b / s[:, :, None]).clamp(-448, 448).to(FP8).view(n, -1)[:, :k]
    return q, s


def check_product(got, a, b, dtype, terms, operand=0.0, bias=None):
    """got against a @ b in 64 bits; `operand`: how far the products' operands may be rounded."""
    ref, size = a @ b, a.abs() @ b.abs()
    if bias is not None:
        ref, size = ref + bias.double(), size + bias.double().abs()
    tol = half_step(dtype) * ref.abs() + ((terms + 4 * -(-terms // 128) + 64) * 2.0 ** -23 * 1.01 + operand) * size
    if dtype == FP16:
        tol = tol + 2.0 ** -25  # half the smallest fp16 step
    assert got.dtype == dtype and got.shape == ref.shape
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), f"{float((off - tol).max())} over, {float((off / tol).nan_to_num().max())} times"


# ---- quantisation -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (2, 129), (5, 16), (7, 1000), (1, 5120), (300, 384),
                                   (2, 3, 250), (100,)])
def test_quantize_is_exact(dtype, shape):
    x = randn(shape, 1, 3.0, dtype)
    q, s = ops.quantize(x)
    ref, ref_s = quantize64(x)
    assert q.dtype == FP8 and q.shape == x.shape and s.shape == (*shape[:-1], -(-shape[-1] // 128))
    assert torch.equal(s.double().reshape(ref_s.shape), ref_s)
    assert torch.equal(values((q, s)).reshape(ref.shape), ref)
    assert torch.equal(ops.dequantize((q, s), dtype).double().reshape(ref.shape), ref)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize_of_views(dtype):
    base = randn((40, 700), 2, 1.0, dtype)
    for v in (base[:, 8:400], base[:, 3:300], base[::2], base[1::3, 5:], base.t(), base[:, :1], base[:0], base[:, ::2]):
        q, s = ops.quantize(v)
        if v.numel() == 0:
            assert q.shape == v.shape
            continue
        ref, ref_s = quantize64(v)
        assert torch.equal(values((q, s)), ref) and torch.equal(s.double(), ref_s)


def test_quantize_borders_and_values_that_are_not_finite():
    f = torch.finfo(FP32)
    x = torch.zeros(12, 256, device="cuda")
    x[1, :128] = f.tiny / 8  # subnormal blocks sit on the smallest scale
    x[2, 0] = f.max
    x[2, 1] = 1.0
    x[3, 0] = math.nan
    x[3, 1] = -2.0
    x[4, 0], x[4, 130] = math.inf, -math.inf
    x[4, 1] = 3.0
    x[5, 0] = 448.0
    x[6, 0] = 448.0000305  # the next fp32 value: one binade more
    x[7, :16] = torch.arange(16, device="cuda") * 2.0 ** -9  # e4m3's subnormals beside 448
    x[7, 20] = 448.0
    x[8, :64] = torch.linspace(-464, 464, 64, device="cuda")
    x[9, 0], x[9, 1], x[9, 2] = 448.0, 17.0, 19.0  # ties: 16 | 18 and 18 | 20
    x[10] = -0.0
    x[11, 255] = 2.0 ** -126
    q, s = ops.quantize(x)
    ref, ref_s = quantize64(x)
    assert torch.equal(s.double(), ref_s)
    got = values((q, s))
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(), ref.nan_to_num())
    assert got[9, 1] == 16 and got[9, 2] == 20 and got[3, 1] == -2
    assert torch.equal(ops.dequantize((q, s), FP32).isnan(), ref.isnan())
    zero = ops.quantize(torch.zeros(3, 300, device="cuda"))
    assert bool((zero[1] == 1).all()) and not values(zero).any()


def test_quantize_writes_nothing_beside_its_rows():
    x = randn((4, 1000), 3)
    (q, s), pitch = ops.block128._empty_pair(x, (4,), 1000)
    base = torch.full((6, pitch), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((6, 8), 7.0, device="cuda")
    ops.block128.native().k_quantize_block128(x.data_ptr(), 1000, 0, base[1:].data_ptr(), pitch, scales[1:].data_ptr(),
                                              4, 1000, torch.cuda.current_stream().cuda_stream)
    assert bool((base[[0, 5]] == 0x55).all()) and bool((base[:, 1000:] == 0x55).all())
    assert bool((scales[[0, 5]] == 7).all())
    q, s = ops.quantize(x)
    assert torch.equal(base[1:5, :1000], q.view(torch.uint8)) and torch.equal(scales[1:5], s)


# ---- the product --------------------------------------------------------------------------------------------------

SHAPES = [(1, 128, 1), (1, 5120, 640), (2, 128, 129), (3, 384, 255), (7, 1792, 1003), (16, 256, 512), (17, 4096, 136),
          (33, 128, 40), (64, 1024, 384), (65, 640, 1000), (128, 512, 256), (129, 256, 257), (200, 3456, 130),
          (256, 384, 512), (300, 2048, 777), (513, 128, 1025), (640, 1280, 2048), (1531, 896, 5001), (2100, 384, 3333),
          (40, 4096, 1000), (100, 2048, 200), (20, 14336, 1024), (12, 5120, 4100)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_linear(m, k, n, dtype):
    x, w = randn((m, k), m, 1.0, dtype), amax_pair(n, k, n)
    bias = randn((n,), 5, 1.0, dtype) if n % 2 else None
    y = ops.linear(x, w, bias)
    check_product(y, quantize64(x)[0], values(w).t(), dtype, k, bias=bias)


@pytest.mark.parametrize("k", [1, 15, 100, 129, 1000])
@pytest.mark.parametrize("m,n", [(1, 7), (40, 200), (150, 300)])
def test_linear_of_ragged_widths(m, n, k):
    x, w = randn((m, k), 1), randn((n, k), 2, 0.1)
    y = ops.linear(x, w, out_dtype=FP32)
    check_product(y, quantize64(x)[0], quantize64(w)[0].t(), FP32, k)


def test_linear_shapes_and_scale_forms():
    x, w = randn((2, 3, 5, 256), 1), amax_pair(72, 256, 2)
    y = ops.linear(x, w)
    assert y.shape == (2, 3, 5, 72)
    flat = ops.linear(x.reshape(-1, 256), (w[0], w[1].reshape(-1)))  # restored weights have flat scales
    assert torch.equal(flat, y.view(-1, 72))
    assert torch.equal(ops.linear(x[1, 2, 4], w), y[1, 2, 4])
    odd = torch.empty(72, 300, dtype=torch.uint8, device="cuda").view(FP8)[:, 3:259]  # rows off the 16-byte grid
    odd.view(torch.uint8).copy_(w[0].view(torch.uint8))
    assert torch.equal(ops.linear(x, (odd, w[1])), y)
    wide = torch.zeros(30, 512, dtype=BF16, device="cuda")
    wide[:, 256:] = x.view(-1, 256)
    assert torch.equal(ops.linear(wide[:, 256:], w), y.view(-1, 72))
    assert torch.equal(ops.linear(x.view(-1, 256).t().contiguous().t(), w), y.view(-1, 72))
    assert ops.linear(x[:0], w).shape == (0, 3, 5, 72)
    assert ops.linear(x, (w[0][:0], w[1][:0])).shape == (2, 3, 5, 0)
    none = ops.linear(x[..., :0], (w[0][:, :0], w[1][:, :0]), torch.ones(72, device="cuda", dtype=BF16))
    assert none.shape == y.shape and bool((none == 1).all())


def test_linear_extremes():
    x = randn((70, 384), 1)
    x[3] = 0
    x[5, 7] = math.nan
    x[6, 200] = math.inf
    w = amax_pair(90, 384, 2)
    w[0].view(torch.uint8)[11] = 0
    w[1][11] = 1
    y = ops.linear(x, w)
    assert not y[3].any() and y[5].isnan().all() and y[6].isnan().all()
    keep = [i for i in range(70) if i not in (5, 6)]
    assert not y[keep, 11].any()
    check_product(y[keep], quantize64(x)[0][keep], values(w).t(), BF16, 384)
    w[0].view(torch.uint8)[4, 9] = 0x7F  # a weight that is not a number spoils its own output alone
    y2 = ops.linear(x, w)
    assert y2[:, 4].isnan().all()
    rest = [j for j in range(90) if j != 4]
    assert torch.equal(y2[keep][:, rest], y[keep][:, rest])
    for scale in (2.0 ** 100, 2.0 ** -100):  # scales whose product is in range although each is far out
        big = (w[0][:4], w[1][:4] * scale)
        got = ops.linear((x[:3].float() / scale).to(BF16), big, out_dtype=FP32)
        check_product(got, quantize64((x[:3].float() / scale).to(BF16))[0], values(big).t(), FP32, 384)


def test_linear_repeats_bit_for_bit():
    for m, k, n in ((1, 5120, 640), (48, 4096, 300), (300, 1024, 512)):
        x, w = randn((m, k), 1), amax_pair(n, k, 2)
        y = ops.linear(x, w)
        assert all(torch.equal(ops.linear(x, w), y) for _ in range(5))


# ---- its gradients ------------------------------------------------------------------------------------------------

GRAD_SHAPES = [(1, 8, 16), (1, 1, 1), (2, 128, 128), (77, 520, 1000), (3, 1003, 257), (128, 256, 384), (130, 72, 40),
               (257, 264, 1001), (64, 2048, 128), (1000, 136, 520), (512, 512, 512), (2051, 130, 260), (5, 4096, 300),
               (1030, 200, 130), (600, 1500, 1400)]


@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
@pytest.mark.parametrize("out", [BF16, FP32])
def test_input_grad(m, n, k, out):
    dy = randn((m, n), 1, 1e-2)
    for w, operand in ((ops.quantize(randn((n, k), 2, 0.05)), 0.0), (amax_pair(n, k, 3), 2.0 ** -8)):
        check_product(ops.linear_input_grad(dy, w, out), dy.double(), values(w), out, n, operand)


@pytest.mark.parametrize("m,n,k", GRAD_SHAPES)
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
def test_weight_grad(m, n, k, out):
    dy, x = randn((m, n), 1, 1e-2), ops.quantize(randn((m, k), 2))
    check_product(ops.linear_weight_grad(dy, x, out), dy.double().t(), values(x), out, m)


@pytest.mark.parametrize("m,n,k", [(20000, 40, 200), (33000, 300, 520), (8192, 64, 128), (8193, 64, 128),
                                   (2049, 600, 3000), (20000, 40, 201)])
def test_long_sums(m, n, k):
    """The tensor core rounds its fp32 additions towards zero, one for each 16 products. They come in runs, of 2048
    products where fp32 results can be stored as tiles and of 8192 elsewhere, and the runs are added to nearest: 128
    (512) units of 2^-23 of the magnitudes' sum for a run, 16 within a step, half a one for each run."""
    units = (128 + 16 + m / 4096 + 1 if k % 4 == 0 else 512 + 16 + m / 16384 + 1) * 2.0 ** -23 * 1.01
    dy, x = randn((m, n), 1, 1.0) + 1, ops.quantize(randn((m, k), 2) + 1)  # a mean, so that errors add up
    a, b = dy.double().t(), values(x)
    got = ops.linear_weight_grad(dy, x, FP32)
    assert bool(((got.double() - a @ b).abs() <= units * (a.abs() @ b.abs())).all())
    assert torch.equal(ops.linear_weight_grad(dy, x, FP32), got)
    got = ops.linear_input_grad(dy.t().contiguous(), x, FP32)
    assert bool(((got.double() - a @ b).abs() <= units * (a.abs() @ b.abs())).all())


@pytest.mark.parametrize("m,n,k", [(1, 4737, 2924), (3, 2000, 1004), (130, 1111, 268)])
def test_many_short_tiles_repeat(m, n, k):
    """Tiles whose sum is a step or two keep the stores behind one another; the last columns of a row fill only the
    first half of a stored piece."""
    dy, x = randn((m, n), 1), ops.quantize(randn((m, k), 2))
    want = ops.linear_weight_grad(dy, x, FP32)
    check_product(want, dy.double().t(), values(x), FP32, m)
    assert all(torch.equal(ops.linear_weight_grad(dy, x, FP32), want) for _ in range(100))


def test_gradients_of_views_and_empty_shapes():
    dy, x = randn((60, 300), 1), ops.quantize(randn((60, 200), 2))
    w = ops.quantize(randn((300, 200), 3))
    dw, dx = ops.linear_weight_grad(dy, x, FP32), ops.linear_input_grad(dy, w, FP32)
    pad = torch.zeros(60, 333, dtype=BF16, device="cuda")
    pad[:, 5:305] = dy
    for v in (pad[:, 5:305], dy.t().contiguous().t(), dy.view(3, 20, 300)):
        assert torch.equal(ops.linear_input_grad(v, w, FP32).view(60, 200), dx)
        assert torch.equal(ops.linear_weight_grad(v, (x[0].view(*v.shape[:-1], 200), x[1]), FP32), dw)
    one = torch.ones(1, 1, dtype=BF16, device="cuda").expand(60, 300)
    check_product(ops.linear_weight_grad(one, x, FP32), one.double().t(), values(x), FP32, 60)
    assert not ops.linear_weight_grad(dy[:0], (x[0][:0], x[1][:0])).any()
    assert ops.linear_input_grad(dy[:0], w).shape == (0, 200)
    assert not ops.linear_input_grad(dy[:, :0], (w[0][:0], w[1][:0])).any()


def test_gradients_repeat_bit_for_bit():
    dy, x, w = randn((2000, 96), 1), ops.quantize(randn((2000, 160), 2)), ops.quantize(randn((96, 160), 3))
    dw, dx = ops.linear_weight_grad(dy, x), ops.linear_input_grad(dy, w)
    for _ in range(5):
        assert torch.equal(ops.linear_weight_grad(dy, x), dw) and torch.equal(ops.linear_input_grad(dy, w), dx)


# ---- the gated activation -----------------------------------------------------------------------------------------

def swiglu64(g, u, dh):
    s = torch.sigmoid(g)
    return g * s * u, dh * u * s * (1 + g * (1 - s)), dh * g * s


def check_swiglu(g, u, dh, dtype):
    """exp in fp32 is off by a few units for each unit of its argument, the rest of the formula by 16."""
    h, kept = ops.swiglu_forward(g, u)
    dg, du = ops.swiglu_backward(dh, kept)
    g64, u64, d = g.double(), u.double(), dh.double()
    kg, ku = quantize64(g)[0].view(g.shape), quantize64(u)[0].view(u.shape)
    assert torch.equal(values(kept[0]), kg) and torch.equal(values(kept[1]), ku)
    s, ks = torch.sigmoid(g64), torch.sigmoid(kg)
    _, rg, ru = swiglu64(kg, ku, d)
    unit, least = (16 + 4 * g64.abs().clamp(max=128)) * 2.0 ** -24, torch.finfo(dtype).tiny
    kunit = (16 + 4 * kg.abs().clamp(max=128)) * 2.0 ** -24
    for got, ref, size, eps in ((h, g64 * s * u64, g64 * s * u64, unit),
                                (dg, rg, d * ku * ks * (1 + kg.abs()), kunit), (du, ru, ru, kunit)):
        tol = half_step(dtype) * ref.abs() + eps * size.abs() + least
        assert got.dtype == dtype and got.shape == ref.shape
        off = (got.double() - ref).abs()
        assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 129), (5, 1000), (64, 3456), (2, 3, 250)])
def test_swiglu(dtype, shape):
    check_swiglu(randn(shape, 1, 2.0, dtype), randn(shape, 2, 1.0, dtype), randn(shape, 3, 1.0, dtype), dtype)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_swiglu_far_out(dtype):
    g = torch.linspace(-200, 200, 4096, device="cuda").to(dtype).view(4, 1024)
    check_swiglu(g, randn((4, 1024), 1, 1.0, dtype), randn((4, 1024), 2, 1.0, dtype), dtype)


def test_swiglu_of_halves_of_one_tensor():
    both = randn((33, 2 * 500), 1, 2.0)
    gate, up = both[:, :500], both[:, 500:]
    h, kept = ops.swiglu_forward(gate, up)
    h2, kept2 = ops.swiglu_forward(gate.contiguous(), up.contiguous())
    assert torch.equal(h, h2)
    d = randn((33, 500), 2)
    assert all(torch.equal(a, b) for a, b in zip(ops.swiglu_backward(d, kept), ops.swiglu_backward(d, kept2)))
    assert ops.swiglu(gate[:0], up[:0]).shape == (0, 500)


def test_swiglu_gradient_against_differences():
    """Central differences of the 64-bit formula at the kept values: their own error is f''' step^2 / 6 < 1e-7 and
    1e-16 |h| / step < 1e-9 of sizes below 20, far under the fp32 gradient's 2^-24 x (16 + 4 |g|)."""
    g, u, d = randn((4, 256), 1, 1.0, FP32), randn((4, 256), 2, 1.0, FP32), randn((4, 256), 3, 1.0, FP32)
    _, kept = ops.swiglu_forward(g, u)
    dg, du = ops.swiglu_backward(d, kept)
    kg, ku, d = values(kept[0]), values(kept[1]), d.double()
    step = 1e-4
    f = lambda a, b: d * swiglu64(a, b, d)[0]  # noqa: E731
    ng = (f(kg + step, ku) - f(kg - step, ku)) / (2 * step)
    nu = (f(kg, ku + step) - f(kg, ku - step)) / (2 * step)
    bound = 32 * 2.0 ** -24 * (1 + kg.abs()) ** 2 * d.abs() * (1 + ku.abs()) + 1e-6
    assert bool(((dg.double() - ng).abs() <= bound).all()) and bool(((du.double() - nu).abs() <= bound).all())


# ---- together -----------------------------------------------------------------------------------------------------

def integers(shape, seed, top=8):
    """Small integers: bfloat16 and the 8-bit form hold them, and differences of them, without a rounding."""
    return torch.randint(-top, top + 1, shape, generator=gen(seed), device="cuda").to(BF16)


def test_linear_gradient_against_differences():
    """y is linear in x and in w: with integers nothing is rounded before the last step, so a difference along any
    integer direction equals the gradient's product with it, up to the gradients' rounding to bfloat16."""
    x, w, dy = integers((37, 300), 1), integers((50, 300), 2), integers((37, 50), 3, 3)
    b = integers((50,), 4)
    xg, wg, bg = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    y = ops.linear(xg, wg, bg)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy)

    def f(x, w, b):
        return (dy.double() * ops.linear(x, w, out_dtype=FP32).double()).sum() + (dy.double() * b.double()).sum()

    for v, grad, at in ((integers(x.shape, 5, 4), dx, lambda t: (x + t, w, b)),
                        (integers(w.shape, 6, 4), dw, lambda t: (x, w + t, b)),
                        (integers(b.shape, 7, 4), db, lambda t: (x, w, b + t))):
        want = f(*at(v)) - f(x, w, b)
        got = (grad.double() * v.double()).sum()
        assert abs(got - want) <= half_step(BF16) * (grad.double() * v.double()).abs().sum()




def test_mlp_step_keeps_eight_bits():
    """gate and up products, gated activation, down product, and the whole backward pass, against the same steps in
    64 bits on the bfloat16 tensors in between."""
    m, h, f = 70, 384, 520
    x = randn((2, 35, h), 1).requires_grad_()
    wg, wu = (randn((f, h), s, 0.05).requires_grad_() for s in (2, 3))
    wd = randn((h, f), 4, 0.05, FP32).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        gate, up = ops.linear(x, wg), ops.linear(x, wu)
        act = ops.swiglu(gate, up)
        y = ops.linear(act, wd)
    big = [t for t in kept if t.numel() >= m * h // 4]
    assert big and all(t.dtype == FP8 for t in big)
    dy = randn(y.shape, 5, 1e-2)
    mid = [gate, up, act]
    grads = torch.autograd.grad(y, (x, wg, wu, wd, *mid), dy, retain_graph=True)
    dx, dwg, dwu, dwd, dgate, dup, dact = grads
    assert dwd.dtype == FP32 and dwg.dtype == BF16 and dx.shape == x.shape
    x2, a2 = (quantize64(t.detach())[0] for t in (x, act))
    qg, qu, qd = (quantize64(t.detach())[0] for t in (wg, wu, wd))
    d = dy.double().reshape(m, h)
    check_product(gate.detach().view(m, f), x2, qg.t(), BF16, h)
    check_product(dact.view(m, f), d, qd, BF16, h)
    check_product(dwd, d.t(), a2, FP32, m)
    check_product(dwg, dgate.double().view(m, f).t(), x2, BF16, m)
    check_product(dwu, dup.double().view(m, f).t(), x2, BF16, m)
    # x feeds two products: autograd adds their two bfloat16 gradients
    a, b = dgate.double().view(m, f), dup.double().view(m, f)
    size = a.abs() @ qg.abs() + b.abs() @ qu.abs()
    parts = (a @ qg).abs() + (b @ qu).abs()
    tol = half_step(BF16) * (parts + (a @ qg + b @ qu).abs()) * 1.01 + (f + 100) * 2.0 ** -23 * size
    assert bool(((dx.double().view(m, h) - a @ qg - b @ qu).abs() <= tol).all())
    again = torch.autograd.grad(y, (x, wg, wu, wd), dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


def test_frozen_pair_passes_gradients_to_the_input_alone():
    x, w = randn((20, 256), 1).requires_grad_(), amax_pair(64, 256, 2)
    b = torch.zeros(64, device="cuda", dtype=BF16).requires_grad_()
    y = ops.linear(x, w, b)
    y.backward(torch.ones_like(y))
    check_product(x.grad, torch.ones(20, 64, device="cuda").double(), values(w), BF16, 64, 2.0 ** -8)
    assert bool((b.grad == 20).all())
    with torch.no_grad():
        assert torch.equal(ops.linear(x, w, b), y)


def test_other_streams_and_captured_graphs():
    x, w = randn((65, 512), 1), amax_pair(200, 512, 2)
    gate = randn((65, 200), 3)
    dy = randn((65, 200), 4)

    def step():
        y = ops.linear(x, w)
        act, kept = ops.swiglu_forward(y, gate)
        return (y, act, *ops.swiglu_backward(dy, kept), ops.linear_input_grad(dy, w),
                ops.linear_weight_grad(dy, ops.quantize(x)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    x0 = x.clone()
    x.copy_(randn((65, 512), 9))
    want2 = step()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want2))
    x.copy_(x0)
    graphs[0][0].replay()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], want))


def test_restored_and_evicted_pairs(sock_path):
    """A weight that comes back from the host in fp8 goes into the product as it is; a checkpoint may leave the GPU
    between the passes."""
    from statespectre_b200 import in_process_daemon, offload_context

    d = in_process_daemon(socket=sock_path, arena_mb=256, drain_on_complete=False)
    try:
        with offload_context(daemon_addr=sock_path, device="cuda:0", rank=0) as off:
            w = randn((640, 1024), 1, 0.02)
            handle = off.copy(w, wait=True)
            pair = handle.restore(cast="fp8_block128")
            x = randn((50, 1024), 2)
            y = ops.linear(x, pair)
            q, s = pair
            check_product(y, quantize64(x)[0], values((q, s.view(640, 8))).t(), BF16, 1024)
            kept = ops.quantize(x)
            dy = randn((50, 640), 3)
            want = ops.linear_weight_grad(dy, kept)
            handles = [off.evict(t, wait=True) for t in kept]
            assert all(t.numel() == 0 for t in kept)
            back = tuple(h.restore() for h in handles)
            assert torch.equal(ops.linear_weight_grad(dy, back), want)
            for h in (*handles, handle):
                h.discard()
    finally:
        d.stop()


def test_rollout_weights_multiply_as_pushed():
    """Weights that a trainer pushed in fp8 go into products where they are, next to parameters that stay bfloat16."""
    from statespectre_b200.parallel.weight_sync import RolloutWeights, WeightLayout, WeightPusher

    params = {"up": randn((640, 512), 1, 0.02), "up.bias": randn((640,), 2), "head": randn((40, 72), 3, 0.1),
              "odd": randn((256, 200), 4, 0.02)}
    layout = WeightLayout.from_params(params, "fp8")
    assert [e.quant for e in layout.entries] == [True, False, False, True]
    rw = RolloutWeights(layout)
    push = WeightPusher(params, layout, rw.buf.data_ptr())
    push.push()
    torch.cuda.synchronize()
    assert push.result()["error"] == 0
    x = randn((33, 512), 5)
    q, s = rw.get("up")
    w64 = values((q, s.view(640, 4)))
    check_product(rw.linear(x, "up", "up.bias"), quantize64(x)[0], w64.t(), BF16, 512, bias=params["up.bias"])
    assert torch.equal(rw.dequantized("up"), w64.to(FP32).to(BF16))
    y = randn((5, 72), 6)
    assert torch.equal(rw.linear(y, "head"), torch.nn.functional.linear(y, params["head"]))
    with pytest.raises(ValueError, match="span rows"):
        rw.linear(randn((5, 200), 7), "odd")
    assert rw.dequantized("odd").shape == (256, 200)


def test_first_call_may_be_captured():
    """A process whose first product runs under graph capture: what the library sets up on a device's first use does
    not break the capture."""
    import subprocess
    import sys

    code = """
import torch
from statespectre_b200 import ops
x = torch.randn(300, 512, device="cuda", dtype=torch.bfloat16)
w = ops.quantize(torch.randn(256, 512, device="cuda"))
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.linear(x, w)
    dx = ops.linear_input_grad(y, w)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, ops.linear(x, w)) and torch.equal(dx, ops.linear_input_grad(y, w))
print("captured")
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120,
                         cwd=__file__.rsplit("/tests/", 1)[0])
    assert "captured" in out.stdout, out.stderr[-2000:]


def test_calls_from_several_threads():
    import threading

    jobs = [(65 + 40 * i, 512, 200 + 64 * i) for i in range(4)]
    data = [(randn((m, k), i), amax_pair(n, k, i + 9), randn((m, n), i + 20, 1e-2)) for i, (m, k, n) in enumerate(jobs)]

    def work(x, w, dy):
        return ops.linear(x, w), ops.linear_input_grad(dy, w), ops.linear_weight_grad(dy, ops.quantize(x))

    want = [work(*d) for d in data]
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = work(*data[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_backward_captured_and_replayed():
    """A training step under capture gives the eager step's gradients, and follows its inputs."""
    m, h, f = 96, 256, 384
    x, dy = randn((m, h), 1), randn((m, h), 5, 1e-2)
    wu, wd = (randn(s, i, 0.05).requires_grad_() for i, s in ((2, (2 * f, h)), (3, (h, f))))

    def step():
        both = ops.linear(x, wu)
        y = ops.linear(ops.swiglu(both[:, :f], both[:, f:]), wd)
        return torch.autograd.grad(y, (wu, wd), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (7, 8):
        x.copy_(randn((m, h), seed))
        g.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_kept_activations_leave_the_gpu_between_the_passes(sock_path):
    """What the forward pass keeps goes to pinned host memory through a session and comes back for the backward pass;
    the gradients are the same bits."""
    from statespectre_b200 import in_process_daemon, offload_context

    m, h, f = 512, 1024, 1536
    x, dy = randn((m, h), 1), randn((m, h), 2, 1e-2)
    wu, wd = (randn(s, i, 0.05).requires_grad_() for i, s in ((3, (2 * f, h)), (4, (h, f))))

    def step():
        both = ops.linear(x, wu)
        return torch.autograd.grad(ops.linear(ops.swiglu(both[:, :f], both[:, f:]), wd), (wu, wd), dy)

    want = step()
    d = in_process_daemon(socket=sock_path, arena_mb=256, drain_on_complete=False)
    try:
        with offload_context(daemon_addr=sock_path, device="cuda:0", rank=0) as off:
            handles = []

            def pack(t):
                if t.dtype != FP8:
                    return t
                handles.append(off.copy(t, wait=True))
                return handles[-1]

            def unpack(k):
                return k if isinstance(k, torch.Tensor) else k.restore()

            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                got = step()
            assert sum(k.nbytes for k in handles) >= m * (h + 3 * f)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for k in handles:
                k.discard()
    finally:
        d.stop()
