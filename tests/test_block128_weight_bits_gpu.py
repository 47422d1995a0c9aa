"""How many bits of an 8-bit operand reach the gradients' products.

A pair's values are e4m3 times any fp32 scale, and only powers of two leave a value that bfloat16 holds. Tolerances: a
value taken to bfloat16 leaves at most 2^-8 of it over, that taken to bfloat16 at most 2^-16, a third part at most 2^-24;
the fp32 product q * scale is off by at most 2^-24. Results in 16 bits take two parts, those in fp32 three. The sums'
bound is the one of test_block128_gpu."""

import pytest
import torch

from statespectre_b200 import ops
from test_block128_gpu import BF16, FP16, FP32, FP8, amax_pair, check_product, gen, half_step, randn, values

pytestmark = pytest.mark.gpu


def off(dtype):
    return 2.0 ** -23 if dtype == FP32 else 2.0 ** -16 + 2.0 ** -24


def mixed_pair(rows, cols, seed, other=0.02):
    """Powers of two as scales, but for a few rows' blocks (`other` of them): steps of the sum with and without them."""
    q, s = ops.quantize(randn((rows, cols), seed, 0.05))
    pick = torch.rand(s.shape, generator=gen(seed + 1), device="cuda") < other
    return q, torch.where(pick, s * (1 + torch.rand(s.shape, generator=gen(seed + 2), device="cuda")), s)


# one CTA on a tile, its sum in parts, pairs of CTAs; short sums, where a term's own error is what is seen
SHAPES = [(5, 1, 300), (33, 3, 129), (64, 8, 1000), (200, 65, 257), (3, 700, 128), (130, 2100, 200), (1300, 3, 1500),
          (1500, 200, 1400), (1100, 1030, 2600)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
def test_input_grad(m, n, k, out):
    dy = randn((m, n), 1, 1.0)
    for w in (amax_pair(n, k, 3), mixed_pair(n, k, 4), mixed_pair(n, k, 5, 0.5)):
        check_product(ops.linear_input_grad(dy, w, out), dy.double(), values(w), out, n, off(out))


@pytest.mark.parametrize("n,m,k", SHAPES)
@pytest.mark.parametrize("out", [BF16, FP16, FP32])
def test_weight_grad(m, n, k, out):
    dy = randn((m, n), 1, 1.0)
    for x in (amax_pair(m, k, 3, 1.0), mixed_pair(m, k, 4)):
        check_product(ops.linear_weight_grad(dy, x, out), dy.double().t(), values(x), out, m, off(out))


@pytest.mark.parametrize("m,n,k", [(256, 2048, 512), (2048, 1536, 1792)])
def test_the_result_is_rounded_once(m, n, k):
    """Over a whole result the error is that of rounding the exact one to bfloat16. What comes before adds in squares:
    2^-16 of each term and truncated additions (n / 16 of them, half a unit of 2^-23 of a partial sum each) are under
    2e-5 where the rounding is 1.6e-3, a part in 5000 of the whole; a part in 100 is granted."""
    dy, w = randn((m, n), 1, 1.0), amax_pair(n, k, 2)
    ref = dy.double() @ values(w)
    got = ops.linear_input_grad(dy, w).double()
    assert (got - ref).norm() <= 1.01 * (ref.to(BF16).double() - ref).norm()


def test_values_past_the_largest_bfloat16():
    """A pair may hold values between the largest bfloat16 and the largest fp32 number; their products are finite."""
    q = torch.zeros(64, 256, device="cuda")
    q[::3, ::2], q[::3, 5], q[7, 3] = 448.0, -416.0, 7.0
    q = q.to(FP8)
    s = torch.full((64, 2), 3.4025e38 / 448, device="cuda")
    dy = randn((40, 64), 1, 2.0 ** -20)
    for out in (BF16, FP32):
        got = ops.linear_input_grad(dy, (q, s), out)
        assert bool(got.isfinite().all())
        check_product(got, dy.double(), values((q, s)), out, 64, off(out))


def test_what_is_not_finite_stays_where_it_is():
    w = amax_pair(300, 256, 2)
    w[1][17, 1] = float("inf")
    w[1][170, 0] = float("nan")
    dy = randn((20, 300), 1)
    clean = (w[0], w[1].nan_to_num(1.0, 1.0))
    dy[3, 17] = 0
    got, want = ops.linear_input_grad(dy, w, FP32), ops.linear_input_grad(dy, clean, FP32)
    assert bool(got[:, :128].isnan().all()) and not bool(got[:, 128:].isfinite().any())
    keep = torch.arange(300, device="cuda") % 7 == 3
    keep[[17, 170]] = False
    part = dy[:, keep].contiguous()
    sub = (w[0][keep].contiguous(), w[1][keep].contiguous())
    check_product(ops.linear_input_grad(part, sub, FP32), part.double(), values(sub), FP32, int(keep.sum()), off(FP32))
    assert want.isfinite().all()


def test_powers_of_two_and_other_scales_repeat_bit_for_bit():
    """Steps with one, two or three tiles of a weight follow one another in the same buffers."""
    for m, n, k, out in ((2100, 1500, 2600, BF16), (2100, 1500, 2600, FP32), (130, 4000, 300, BF16), (77, 9000, 520, FP32)):
        dy, w = randn((m, n), 1), mixed_pair(n, k, 2, 0.01)
        want = ops.linear_input_grad(dy, w, out)
        check_product(want, dy.double(), values(w), out, n, off(out))
        assert all(torch.equal(ops.linear_input_grad(dy, w, out), want) for _ in range(40))


def test_gradient_at_the_weights_that_the_product_saw():
    """The gradient of a product with a pushed or restored weight: dy @ w at the pair's own values."""
    x, w = randn((150, 384), 1).requires_grad_(), amax_pair(640, 384, 2)
    y = ops.linear(x, w)
    dy = randn((150, 640), 3)
    dx, = torch.autograd.grad(y, x, dy)
    check_product(dx, dy.double(), values(w), BF16, 640, off(BF16))
    ref = dy.double() @ values(w)
    assert (dx.double() - ref).norm() <= 1.01 * (ref.to(BF16).double() - ref).norm()
    assert half_step(BF16) == 2.0 ** -8


def test_captured_gradients_follow_their_scales():
    """The kind of a pair's scales is found as the work runs: graphs that replay side by side, in pairs of CTAs and in
    single ones, give what eager calls give as powers of two turn into other scales and back."""
    cases = [(randn((1300, 520), 1), amax_pair(520, 1500, 2)), (randn((70, 900), 3), amax_pair(900, 300, 4)),
             (randn((600, 1400), 5), amax_pair(1400, 2600, 6))]
    both = [(s, 2.0 ** torch.floor(torch.log2(s))) for _, (_, s) in cases]
    both = [(a.clone(), b) for a, b in both]

    def step():
        return [ops.linear_input_grad(dy, w, out) for dy, w in cases for out in (BF16, FP32)]

    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out, torch.cuda.Stream()))
    for turn in range(6):
        for (_, w), kinds in zip(cases, both):
            w[1].copy_(kinds[turn % 2])
        want = step()
        for g, _, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for _, out, s in graphs:
            torch.cuda.current_stream().wait_stream(s)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    i = 0
    for dy, w in cases:
        for out in (BF16, FP32):
            check_product(want[i], dy.double(), values(w), out, dy.shape[1], off(out))
            i += 1


def test_pairs_of_several_threads():
    import threading

    data = [(randn((700 + 200 * i, 300 + 64 * i), i), amax_pair(300 + 64 * i, 2600, i + 9)) for i in range(3)]
    want = [ops.linear_input_grad(*d) for d in data]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = ops.linear_input_grad(*data[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
