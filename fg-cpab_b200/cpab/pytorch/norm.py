"""Root-mean-square norm with the residual's addition, and its 8-bit form.

    s = x + residual,   y = s / sqrt(mean(s^2) + eps) * weight    (last axis)

s is rounded to the residual's type and is what the next block adds to; y is
the norm of what was kept.  No counterpart in the reference.
"""
import torch

from .. import _ext, _native


def rms_norm(x, weight, residual=None, eps=1e-6):
    """x [..., D] float32, float16 or bfloat16 (D at most 16384); weight [D]
    and residual [..., D] of x's type or float32.  Returns y (x's type), or
    (y, s) with a residual (s of the residual's type).  Differentiable (once)
    in x, weight and residual, backward only."""
    ext = _ext.module()
    if ext is None:
        _native.check_norm(x, weight, residual)
        if _native.needs_grad(x, weight, residual):
            out = _RmsNorm.apply(x, weight, residual, float(eps))
        else:
            out = _native.rms_norm(x, weight, residual, float(eps), False)[:2]
        return out[0] if residual is None else tuple(out)
    out = _ext.call(ext.rms_norm, x, weight, residual, float(eps))
    return out[0] if residual is None else tuple(out)


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, s, rstd = _native.rms_norm(x, weight, residual, eps, True)
        ctx.save_for_backward(x if s is None else s, weight, rstd)
        ctx.x_type, ctx.residual = x.dtype, residual is not None
        ctx.set_materialize_grads(False)
        return (y,) if s is None else (y, s)

    @staticmethod
    def backward(ctx, gy, gs=None):
        if torch.is_grad_enabled():
            raise RuntimeError("rms_norm can be differentiated once only (create_graph=True)")
        s, weight, rstd = ctx.saved_tensors
        if gy is None:
            return (gs.to(ctx.x_type) if gs is not None else None), None, gs, None
        dx, dres, dw = _native.rms_norm_backward(s, weight, rstd, gy, gs, ctx.x_type,
                                                 ctx.needs_input_grad[1])
        return dx, dw, (dres if ctx.residual else None), None


def rms_norm_quantized(x, weight, residual=None, eps=1e-6):
    """rms_norm with y in 8 bits, for networks that answer: (q, scale), or
    (q, scale, s) with a residual, where q [..., D] float8_e4m3fn and scale
    [...] float32 (one per row) stand for y ~ q * scale; scale =
    max(max|y| / 448, 2^-126), never 0.  No gradient."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm_quantized has no gradient; call it under torch.no_grad()")
    ext = _ext.module()
    if ext is None:
        _native.check_norm(x, weight, residual)
        return _native.rms_norm_quantized(x, weight, residual, float(eps))
    return tuple(_ext.call(ext.rms_norm_quantized, x, weight, residual, float(eps)))
