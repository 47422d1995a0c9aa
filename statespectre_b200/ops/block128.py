"""Operators on fp8 block-128 tensors.

A block-128 tensor is the pair ``(q, scales)`` that ``quantize`` makes: ``q`` holds e4m3 values, ``scales`` one
fp32 factor for each 128 consecutive values of a row, [..., ceil(cols / 128)], and the pair stands for
``q * scale``. A row whose length is no multiple of 128 ends in a shorter block of its own, and rows of ``q``
start on 16-byte boundaries (a pair laid out otherwise is copied). ``handle.restore(cast="fp8_block128")`` and
``RolloutWeights.get`` return the same with flat scales where rows are multiples of 128 values; for other widths
their blocks run on from row to row, and the operators refuse the pair.

* ``quantize`` / ``dequantize``: an activation to 8 bits and back, with power-of-two scales
* ``linear``: ``x @ w.T`` on the fp8 tensor cores; with gradients, the quantised operands of the forward
  product are the only activations and weights kept for the backward pass
* ``linear_input_grad`` / ``linear_weight_grad``: the two products of that backward pass
* ``swiglu`` (and its two passes): the gated activation, keeping its inputs in 8 bits

Everything runs on the current stream of the tensors' device and can be captured into a CUDA graph.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from .._native import native

Block128 = Tuple[torch.Tensor, torch.Tensor]

BLOCK = 128
_MOST = 1 << 31  # a row pitch from here on is copied away
_FP8 = torch.float8_e4m3fn
_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


# The current stream and device as plain numbers: torch.cuda's functions build
# objects, which at the smallest sizes takes longer than the kernels.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _type(dtype: torch.dtype, what: str) -> int:
    code = _TYPE.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be bfloat16, float16 or float32; got {dtype}")
    return code


def _on_gpu(t, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor; got {type(t).__name__}")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} has a tangent, and the operators have no forward-mode derivatives")
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t


def _same_device(first: torch.Tensor, t: torch.Tensor, what: str) -> None:
    if t.get_device() != first.get_device():
        raise ValueError(f"{what} is on {t.device}, the first operand on {first.device}")


def _launch(device: int, fn, *args) -> None:
    """``fn(*args, stream)`` on the device's current stream, with the device current."""
    if device == _current_device():
        fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            fn(*args, _raw_stream(device))


def _matrix(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(2-D form with unit column stride, rows, cols, pitch): a view where the strides allow one."""
    if t.dim() != 2:
        if t.dim() == 0:
            raise ValueError(f"{what} must have at least one dimension")
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    rows, cols = t.shape
    pitch, one = t.stride()
    if (cols > 1 and one != 1) or (rows > 1 and not cols <= pitch < _MOST):
        t = t.contiguous()
        pitch = cols
    return t, rows, cols, pitch if rows > 1 else cols


def _tiled(t: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """``_matrix`` whose base and pitch are multiples of 16 bytes, as the tile copies need: a copy if they are not."""
    t, rows, cols, ld = _matrix(t, what)
    per = 16 // t.element_size()
    if rows == 1:
        ld = -(-cols // per) * per
    if ld % per or t.data_ptr() % 16:
        ld = -(-cols // per) * per
        p = torch.empty((rows, ld), dtype=t.dtype, device=t.device)[:, :cols]
        t = p.copy_(t)
    return t, rows, cols, ld


def _constant(p, what: str):
    """The pair's two tensors, checked to want no derivative."""
    if not isinstance(p, (tuple, list)) or len(p) != 2:
        raise TypeError(f"{what} must be a (q, scales) pair")
    q, scales = p
    _on_gpu(q, what)
    _on_gpu(scales, what)
    if (q.requires_grad or scales.requires_grad) and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and a pair has none: detach() it, or call under no_grad()")
    return q, scales


def _row_wise(shape, rows: int, cols: int) -> bool:
    """Whether as many scales as there are blocks lie row by row in this shape: its last dimensions make up a row, or it
    is flat. Flat scales count on from one row to the next, which is the same where rows end on a block."""
    blocks, n = -(-cols // BLOCK), 1
    for d in reversed(shape):
        n *= d
        if n == blocks:
            return True
    return n == 0 or ((rows == 1 or cols % BLOCK == 0) and max(shape, default=1) == n)


def _pair(p, what: str):
    """(q, scales, rows, cols, pitch) of a block-128 pair."""
    q, scales = _constant(p, what)
    if q.dtype != _FP8:
        raise ValueError(f"{what}: q must be float8_e4m3fn; got {q.dtype}")
    if scales.dtype != torch.float32:
        raise ValueError(f"{what}: scales must be float32; got {scales.dtype}")
    _same_device(q, scales, what)
    q, rows, cols, ld = _tiled(q, what)
    blocks = -(-cols // BLOCK)
    if scales.numel() != rows * blocks or not (scales.shape[-1:] == (blocks,) or _row_wise(scales.shape, rows, cols)):
        raise ValueError(f"{what}: {tuple(scales.shape)} scales do not fit {rows} rows of {cols} values: one for "
                         f"each {BLOCK} values of a row, flat only where rows are multiples of {BLOCK}")
    return q, scales if scales.is_contiguous() else scales.contiguous(), rows, cols, ld


def _empty_pair(like: torch.Tensor, lead, cols: int):
    """Uninitialised (q, scales) of [*lead, cols] values, and q's pitch."""
    pitch = -(-cols // 16) * 16
    q = like.new_empty((*lead, pitch), dtype=_FP8)
    if pitch != cols:
        q = q[..., :cols]
    return (q, like.new_empty((*lead, -(-cols // BLOCK)), dtype=torch.float32)), pitch


def _empty_rows(like: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of `like`'s shape and type."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def quantize(x: torch.Tensor) -> Block128:
    """``x`` [..., cols] (bfloat16, float16 or float32) in 8 bits: ``(q, scales)``, ``q`` [..., cols] and one scale
    per 128 values, [..., ceil(cols / 128)].

    The scale is the smallest power of two (at least 2^-117) that brings a block within e4m3's 448, 1 for a block
    of zeros, so the only rounding is e4m3's (to nearest, ties to even). A value that is not finite becomes NaN and
    does not count in its block's scale."""
    _on_gpu(x, "x")
    code = _type(x.dtype, "x")
    lead = x.shape[:-1]
    x, rows, cols, ld = _matrix(x, "x")
    (q, scales), pitch = _empty_pair(x, lead, cols)
    _launch(x.get_device(), native().k_quantize_block128, x.data_ptr(), ld, code, q.data_ptr(), pitch,
            scales.data_ptr(), rows, cols)
    return q, scales


def dequantize(x: Block128, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that a pair stands for, rounded to ``dtype`` (no rounding in bfloat16 and float32 where
    ``quantize`` made the pair)."""
    code = _type(dtype, "dtype")
    q, scales, rows, cols, ld = _pair(x, "x")
    out = q.new_empty(x[0].shape, dtype=dtype)
    _launch(q.get_device(), native().k_dequantize_block128, q.data_ptr(), ld, scales.data_ptr(), out.data_ptr(), cols,
            code, rows, cols)
    return out


def linear(x: torch.Tensor, weight, bias: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``x @ weight.T (+ bias)``: ``x`` [..., k] is quantised (as ``quantize`` does) and multiplied in 8 bits with
    fp32 sums. ``weight`` is a pair [n, k] as restored or pushed in fp8 (any scales), or a floating tensor [n, k],
    which is quantised too. The result has ``x``'s dtype unless ``out_dtype`` says otherwise.

    With gradients (``x`` bfloat16), the backward pass uses the quantised operands: ``dx = dy @ w`` and
    ``dw = dy.T @ x`` at the values that the forward product saw, and nothing else is kept. The quantisation
    itself passes gradients through unchanged."""
    _on_gpu(x, "x")
    _type(x.dtype, "x")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    _type(out_dtype, "out_dtype")
    if isinstance(weight, torch.Tensor):
        _on_gpu(weight, "weight")
        _type(weight.dtype, "weight")
        wanted = x.requires_grad or weight.requires_grad
    else:
        wanted = x.requires_grad
    if bias is not None:
        _on_gpu(bias, "bias")
        wanted = wanted or bias.requires_grad
    if wanted and torch.is_grad_enabled():
        if x.dtype != torch.bfloat16 or out_dtype != torch.bfloat16:
            raise ValueError("linear with gradients needs bfloat16 activations")
        if isinstance(weight, torch.Tensor):
            return _Linear.apply(x, weight, bias, None)
        _constant(weight, "weight")  # here, since the pass itself runs without gradients
        return _Linear.apply(x, None, bias, weight)
    return _forward(x, weight, bias, out_dtype, False)[0]


def _weight_pair(weight):
    q = weight if isinstance(weight, torch.Tensor) else weight[0] if isinstance(weight, (tuple, list)) else None
    if isinstance(q, torch.Tensor) and q.dim() != 2:
        raise ValueError(f"weight must have two dimensions; got {q.dim()}")
    return _pair(quantize(weight) if isinstance(weight, torch.Tensor) else weight, "weight")


def _forward(x, weight, bias, out_dtype, keep: bool):
    """(result, x's pair in two dimensions or None, the weight's pair)."""
    wq, ws, n, k, ldw = wp = _weight_pair(weight)
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"x has shape {tuple(x.shape)}, the weight {k} columns")
    lead = x.shape[:-1]
    x, m, _, ldx = _matrix(x, "x")
    _same_device(x, wq, "weight")
    if bias is not None:
        _same_device(x, bias, "bias")
        if bias.shape != (n,):
            raise ValueError(f"bias must have shape ({n},); got {tuple(bias.shape)}")
        if bias.dtype != out_dtype:
            raise ValueError(f"bias must be {out_dtype} like the result; got {bias.dtype}")
        bias = bias.contiguous()
    y = x.new_empty((*lead, n), dtype=out_dtype)
    if k == 0:
        return (y.zero_() if bias is None else y.copy_(bias.expand_as(y))), quantize(x) if keep else None, wp
    C = native()
    work_bytes = C.linear_work_bytes(m, k)
    pitch = -(-k // 16) * 16
    if keep:
        (q, scales), pitch = _empty_pair(x, (m,), k)
        work = x.new_empty(work_bytes, dtype=torch.uint8)
        ptrs = q.data_ptr(), pitch, scales.data_ptr(), work.data_ptr()
    else:
        work = x.new_empty(work_bytes + m * pitch, dtype=torch.uint8)
        ptrs = work.data_ptr() + work_bytes, pitch, 0, work.data_ptr()
    _launch(x.get_device(), C.k_linear_block128, x.data_ptr(), ldx, _TYPE[x.dtype], *ptrs, work_bytes, wq.data_ptr(),
            ldw, ws.data_ptr(), 0 if bias is None else bias.data_ptr(), y.data_ptr(), n, _TYPE[out_dtype], m, n, k)
    return y, (q, scales) if keep else None, wp


def _gradient(dy: torch.Tensor, other: Block128, what: str):
    _on_gpu(dy, "dy")
    if dy.dtype != torch.bfloat16:
        raise ValueError(f"dy must be bfloat16; got {dy.dtype}")
    p = _pair(other, what)
    _same_device(dy, p[0], what)
    return _tiled(dy, "dy"), p


def _launch_grad(fn, d, ldd, q, ld, scales, out, code, m, n, k, out_rows) -> None:
    device = d.get_device()
    if device == _current_device():
        words = native().grad_work_words(out_rows, k)
        work = d.new_empty(words, dtype=torch.int32) if words else None
        fn(d.data_ptr(), ldd, q.data_ptr(), ld, scales.data_ptr(), out.data_ptr(), k, code, m, n, k,
           _raw_stream(device), work.data_ptr() if words else 0, words)
    else:
        with torch.cuda.device(device):
            _launch_grad(fn, d, ldd, q, ld, scales, out, code, m, n, k, out_rows)


def linear_input_grad(dy: torch.Tensor, weight: Block128, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dy @ w`` for ``dy`` [..., n] (bfloat16) and a pair ``weight`` [n, k]: [..., k]. Each weight goes to the tensor
    cores exactly where its scale is a power of two, else within 2^-16 of it (2^-24 for an fp32 result), which takes
    two (three) products instead of one; sums are in fp32."""
    code = _type(out_dtype, "out_dtype")
    (d, m, n, ldd), (q, scales, rows, k, ld) = _gradient(dy, weight, "weight")
    if rows != n or weight[0].dim() != 2:
        raise ValueError(f"dy has {n} columns, the weight shape {tuple(weight[0].shape)}")
    dx = d.new_empty((*dy.shape[:-1], k), dtype=out_dtype)
    if n == 0:
        return dx.zero_()
    _launch_grad(native().k_matmul_input_grad, d, ldd, q, ld, scales, dx, code, m, n, k, m)
    return dx


def linear_weight_grad(dy: torch.Tensor, x: Block128, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dy.T @ x`` for ``dy`` [..., n] (bfloat16) and the kept pair ``x`` [..., k]: [n, k], summed over all rows in
    fp32. The kept values go to the tensor cores exactly where their scales are powers of two, as ``quantize`` makes
    them, else as in ``linear_input_grad``."""
    code = _type(out_dtype, "out_dtype")
    (d, m, n, ldd), (q, scales, rows, k, ld) = _gradient(dy, x, "x")
    if rows != m:
        raise ValueError(f"dy has {m} rows, x {rows}")
    dw = d.new_empty((n, k), dtype=out_dtype)
    if m == 0:
        return dw.zero_()
    _launch_grad(native().k_matmul_weight_grad, d, ldd, q, ld, scales, dw, code, m, n, k, n)
    return dw


def product_error(device=None, clear: bool = False) -> int:
    """0, or the code of the first product on ``device`` (the current one) whose bounded wait for a tile ran out, which
    leaves its result incomplete. Products launched later raise ``RuntimeError`` for it; a replayed graph and work that
    is still running cannot, so ask after a synchronization. ``clear`` ends the raising."""
    index = None if device is None else torch.device(device).index if not isinstance(device, int) else device
    if index is None:
        index = torch.cuda.current_device()
    code = native().block128_error(index)
    if clear and code:
        native().block128_set_error(index, 0)
    return code


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, pair):
        need_dw = weight is not None and weight.requires_grad
        y, xp, wp = _forward(x, pair if weight is None else weight, bias, torch.bfloat16, need_dw)
        ctx.save_for_backward(*(xp if need_dw else (None, None)),
                              *(wp[:2] if x.requires_grad else (None, None)))
        ctx.x_shape = x.shape
        ctx.weight_dtype = None if weight is None else weight.dtype
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        xq, xs, wq, ws = ctx.saved_tensors
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            dx = linear_input_grad(dy, (wq, ws)).view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            dw = linear_weight_grad(dy, (xq, xs), ctx.weight_dtype)
        if ctx.needs_input_grad[2]:
            db = dy.reshape(dy.shape[:-1].numel(), dy.shape[-1]).sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        return dx, dw, db, None


def swiglu_forward(gate: torch.Tensor, up: torch.Tensor):
    """``silu(gate) * up`` and what its backward pass keeps: ``(h, (kept_gate, kept_up))``, two pairs as ``quantize``
    makes them. ``h`` is computed from the unquantised inputs."""
    _on_gpu(gate, "gate")
    _on_gpu(up, "up")
    code = _type(gate.dtype, "gate")
    shape = gate.shape
    if up.dtype != gate.dtype or up.shape != shape:
        raise ValueError(f"up ({tuple(up.shape)}, {up.dtype}) must match gate ({tuple(shape)}, {gate.dtype})")
    _same_device(gate, up, "up")
    g, rows, cols, ldg = _matrix(gate, "gate")
    u, _, _, ldu = _matrix(up, "up")
    h = _empty_rows(gate)
    kg, pitch = _empty_pair(g, shape[:-1], cols)
    if pitch == cols:
        ku = torch.empty_like(kg[0]), torch.empty_like(kg[1])
    else:
        ku, _ = _empty_pair(g, shape[:-1], cols)
    _launch(g.get_device(), native().k_swiglu_forward, g.data_ptr(), ldg, u.data_ptr(), ldu, code, h.data_ptr(), cols,
            kg[0].data_ptr(), kg[1].data_ptr(), ku[0].data_ptr(), ku[1].data_ptr(), pitch, rows, cols)
    return h, (kg, ku)


def swiglu_backward(dh: torch.Tensor, kept) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(dgate, dup)`` from ``dh`` and what ``swiglu_forward`` kept: the gradients of ``silu(gate) * up`` at the
    kept values, in ``dh``'s dtype."""
    _on_gpu(dh, "dh")
    code = _type(dh.dtype, "dh")
    if not isinstance(kept, (tuple, list)) or len(kept) != 2:
        raise TypeError("kept must be the two pairs that swiglu_forward returned")
    gq, gs, rows, cols, ldg = _pair(kept[0], "kept gate")
    uq, us, rows_u, cols_u, ldu = _pair(kept[1], "kept up")
    d, rows_d, cols_d, ldd = _matrix(dh, "dh")
    if (rows, cols) != (rows_u, cols_u) or (rows, cols) != (rows_d, cols_d):
        raise ValueError(f"dh has shape {tuple(dh.shape)}, the kept pairs {tuple(kept[0][0].shape)} and "
                         f"{tuple(kept[1][0].shape)}")
    _same_device(d, gq, "kept gate")
    _same_device(d, uq, "kept up")
    dg, du = _empty_rows(dh), _empty_rows(dh)
    _launch(d.get_device(), native().k_swiglu_backward, d.data_ptr(), ldd, code, gq.data_ptr(), ldg, gs.data_ptr(),
            uq.data_ptr(), ldu, us.data_ptr(), dg.data_ptr(), du.data_ptr(), cols, rows, cols)
    return dg, du


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        h, (kg, ku) = swiglu_forward(gate, up)
        ctx.save_for_backward(*kg, *ku)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        gq, gs, uq, us = ctx.saved_tensors
        return swiglu_backward(dh, ((gq, gs), (uq, us)))


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up``; with gradients, the inputs are kept in 8 bits (2 bytes a pair of values instead of 4 or
    8) and the backward pass takes its derivatives at the kept values."""
    if torch.is_grad_enabled() and (getattr(gate, "requires_grad", False) or getattr(up, "requires_grad", False)):
        return _SwiGLU.apply(gate, up)
    return swiglu_forward(gate, up)[0]
