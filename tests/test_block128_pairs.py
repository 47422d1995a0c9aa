"""Which scales fit a q: per-row blocks, or the flat scales of a restored tensor where its rows end on a block. Others
have the right number of scales for some shapes and would give wrong values."""

import pytest
import torch

from statespectre_b200 import ops
from statespectre_b200.ops import block128

FP8 = torch.float8_e4m3fn


@pytest.fixture
def any_device(monkeypatch):
    monkeypatch.setattr(block128, "_on_gpu", lambda t, what: t)


def q(*shape):
    return torch.zeros(*shape, dtype=FP8)


# the scales run on across rows, and are as many as one for each 128 values of a row
RUN_ON = [(4, 1000), (64, 1023), (100, 127), (2, 255), (2, 100), (127, 14335)]


@pytest.mark.parametrize("rows,cols", RUN_ON)
@pytest.mark.parametrize("call", [
    lambda p: ops.dequantize(p), lambda p: ops.linear(torch.zeros(2, p[0].shape[1], dtype=torch.bfloat16), p),
    lambda p: ops.linear_input_grad(torch.zeros(2, p[0].shape[0], dtype=torch.bfloat16), p),
    lambda p: ops.linear_weight_grad(torch.zeros(p[0].shape[0], 2, dtype=torch.bfloat16), p),
    lambda p: ops.swiglu_backward(torch.zeros(p[0].shape, dtype=torch.bfloat16), (p, p))])
def test_scales_that_run_on_across_rows_are_refused(any_device, rows, cols, call):
    scales = torch.ones((rows * cols + 127) // 128)
    assert scales.numel() == rows * -(-cols // 128)
    with pytest.raises(ValueError, match="do not fit"):
        call((q(rows, cols), scales))


@pytest.mark.parametrize("shape,scales", [((8, 256), (2, 8)), ((8, 200), (16,)),
                                          ((8, 200), (1, 16)), ((3, 20, 200), (120,)), ((3, 20, 256), (3, 2, 20)),
                                          ((6, 127), (1, 6))])
def test_scales_of_another_shape_are_refused(any_device, shape, scales):
    with pytest.raises(ValueError, match="do not fit"):
        ops.dequantize((q(*shape), torch.ones(scales)))


@pytest.mark.parametrize("shape,scales", [((8, 256), (8, 2)), ((8, 256), (16,)), ((8, 256), (1, 16)), ((8, 256), (16, 1)),
                                          ((8, 256), (8, 2, 1)), ((8, 200), (8, 2, 1)), ((8, 200), (8, 2)), ((1, 100), ()),
                                          ((1, 200), (2,)), ((200,), (2,)), ((3, 20, 200), (3, 20, 2)),
                                          ((3, 20, 200), (60, 2)),
                                          ((60, 200), (3, 20, 2)), ((3, 20, 256), (120,)), ((6, 127), (6, 1)),
                                          ((0, 200), (0, 2)), ((0, 200), (0,)), ((5, 0), (5, 0)), ((1, 1, 200), (2,))])
def test_scales_that_fit(any_device, shape, scales):
    _, s, rows, cols, _ = block128._pair((q(*shape), torch.ones(scales)), "x")
    assert s.numel() == rows * -(-cols // 128) and cols == shape[-1]


@pytest.mark.gpu
def test_a_restored_weight_whose_rows_end_inside_a_block(sock_path):
    from statespectre_b200 import in_process_daemon, offload_context

    d = in_process_daemon(socket=sock_path, arena_mb=64, drain_on_complete=False)
    try:
        with offload_context(daemon_addr=sock_path, device="cuda:0", rank=0) as off:
            w = torch.randn(4, 1000, device="cuda").to(torch.bfloat16)
            handle = off.copy(w, wait=True)
            pair = handle.restore(cast="fp8_block128")
            with pytest.raises(ValueError, match="do not fit"):
                ops.linear(torch.randn(3, 1000, device="cuda").to(torch.bfloat16), pair)
            with pytest.raises(ValueError, match="do not fit"):
                ops.dequantize(pair)
            handle.discard()
    finally:
        d.stop()
