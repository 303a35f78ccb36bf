"""Projections in 8 bits: e4m3 codes with a power-of-two scale for each 128 of
them along the summed axis, their products, and a differentiable projection
made of them.

    s = 2^ceil(log2(max|x| / 448)) >= 2^-126,   q = e4m3(x / s)       (per block)
    y = sum over blocks of (q_x q_w) s_x s_w + bias                    (in float32)

No counterpart in the reference.
"""
import functools

import torch

from .. import _ext, _native


def quantize_blocks(x, transposed=False):
    """x [..., K] float32, float16 or bfloat16 -> (q [..., K] float8_e4m3fn,
    scale [..., ceil(K / 128)] float8_e8m0fnu), x ~ q * scale; rows of q begin
    on multiples of 16 bytes.  transposed=True (x [R, K]): (q, scale, qt,
    scale_t), the last two those of x's transpose, whose blocks run along R.

    A block that holds an infinity or a NaN has the scale NaN.  No gradient."""
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("quantize_blocks has no gradient; call it under torch.no_grad(), or use "
                           "linear_quantized")
    ext = _ext.module()
    if ext is not None:
        return tuple(_ext.call(ext.quantize_blocks, x, bool(transposed)))
    _native.check_quantize(x)
    if _native.has_tangent(x):
        raise RuntimeError("quantize_blocks has no gradient, of forward mode neither")
    if transposed and x.dim() != 2:
        raise ValueError("x must be [R, K] for its transpose, got %s" % (tuple(x.shape),))
    out = _native.quantize_blocks(x, True, transposed)
    return out[:4] if transposed else out[:2]


def matmul_quantized(q, scale, weight, weight_scale, bias=None, dtype=torch.bfloat16):
    """q [..., K] float8_e4m3fn and weight [N, K] float8_e4m3fn -> [..., N] of
    dtype (float32, float16 or bfloat16).  A scale is float8_e8m0fnu
    [..., ceil(K / 128)] (of quantize_blocks) or float32 [...], one for each row
    (of rms_norm_quantized); bias [N] is float32 or of dtype.  Codes whose rows
    do not begin on multiples of 16 bytes are copied.  No gradient (scales,
    codes or a bias that want one are refused)."""
    if torch.is_grad_enabled() and (scale.requires_grad or weight_scale.requires_grad or q.requires_grad or
                                    weight.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("matmul_quantized has no gradient; call it under torch.no_grad(), or use "
                           "linear_quantized")
    ext = _ext.module()
    if ext is None:
        return _native.matmul_quantized(q, scale, weight, weight_scale, bias, dtype)
    return _ext.call(ext.matmul_quantized, q, scale, weight, weight_scale, bias, dtype)


def linear_quantized(x, weight, bias=None):
    """x [..., K] @ weight [N, K]^T + bias [N] with all three products of a
    training step in 8 bits: the output's, the input's gradient's and the
    weight's gradient's operands go through quantize_blocks, each along the axis
    that its product sums.  x float32, float16 or bfloat16; weight and bias of
    x's type or float32.  Differentiable (once, backward only) in x, weight and
    bias, as if the codes were the values."""
    ext = _ext.module()
    if ext is not None:
        return _ext.call(ext.linear_quantized, x, weight, bias)
    _native.check_linear(x, weight, bias)
    if _native.needs_grad(x, weight, bias):
        return _LinearQuantized.apply(x, weight, bias)
    q, s = _native.quantize_blocks(x)[:2]
    w, ws = _native.quantize_blocks(weight)[:2]
    return _native.matmul_quantized(q, s, w, ws, bias, x.dtype)


class _LinearQuantized(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        want_x, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        q, s, qt, st, _ = _native.quantize_blocks(x, True, want_w)
        w, ws, wt, wst, _ = _native.quantize_blocks(weight, True, want_x)
        ctx.save_for_backward(qt, st, wt, wst)
        ctx.K = x.shape[-1]
        ctx.types = x.dtype, weight.dtype, bias.dtype if bias is not None else None
        return _native.matmul_quantized(q, s, w, ws, bias, x.dtype)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("linear_quantized can be differentiated once only (create_graph=True)")
        qt, st, wt, wst = ctx.saved_tensors
        x_type, w_type, b_type = ctx.types
        want_x, want_w, want_b = ctx.needs_input_grad
        if dy.shape[-1] == 0:
            zeros = functools.partial(torch.zeros, device=dy.device)
            return (zeros((*dy.shape[:-1], ctx.K), dtype=x_type) if want_x else None,
                    zeros((0, ctx.K), dtype=w_type) if want_w else None,
                    zeros(0, dtype=b_type) if want_b else None)
        q, s, dt, dst, db = _native.quantize_blocks(dy, want_x, want_w, b_type if want_b else None)
        dx = _native.matmul_quantized(q, s, wt, wst, None, x_type) if want_x else None
        dw = None
        if want_w and dt.shape[1]:
            dw = _native.matmul_quantized(dt, dst, qt, st, None, w_type)
        elif want_w:
            dw = torch.zeros((dt.shape[0], qt.shape[0]), device=dy.device, dtype=w_type)
        return dx, dw, db
