"""The gated linear recurrence over time: the sequence layer of networks that
predict theta from long signals.

    h_t = a_t h_{t-1} + (1 - a_t) x_t,   a_t = sigmoid(gate_t)      (per channel)

gated_scan runs it over whole series, differentiably; gated_scan_step takes
one sample of each of many running streams.  The state is float32 whatever
the inputs' type.  No counterpart in the reference.
"""
import torch

from .. import _ext, _native


def _int32(t, name, most):
    """A vector of whole numbers as int32; 64-bit values are clamped first
    (anything outside [-1, most] means what its bound means)."""
    if t is None or t.dtype == torch.int32:
        return t
    if t.dtype != torch.int64:
        raise TypeError("%s must be int32 or int64, got %s" % (name, t.dtype))
    return t.clamp(-1, most).to(torch.int32)


def gated_scan(x, gate=None, h0=None, lengths=None):
    """The recurrence over x [B, T, D] with gate logits gate [B, T, D], both
    float32, float16 or bfloat16; without gate, x is [B, T, 2 D], a projection
    whose first D channels are the inputs and the others the logits (its
    gradient then comes as one tensor too).  h0 [B, D] float32 is the state
    before the first sample (zeros).  lengths [B] (int32 or int64): series b
    has lengths[b] samples; what x and gate hold after them is never read,
    h is 0 there and the state stays.

    A NaN stays in its channel from its sample on; an infinity does too, as an
    infinity or a NaN.

    Returns (h [B, T, D] of x's type, last [B, D] float32, the state after
    each series' last sample).  Differentiable (once, backward only) in x,
    gate and h0; any strides, without a copy where the channels are adjacent."""
    lengths = _int32(lengths, "lengths", x.shape[1] if x.dim() > 1 else 0)
    ext = _ext.module()
    if ext is None:
        _native.check_scan(x, gate, h0, lengths)
        if _native.needs_grad(x, gate, h0):
            return _GatedScan.apply(x, gate, h0, lengths)
        return _native.gated_scan(x, gate, h0, lengths, False)[:2]
    return _ext.call(ext.gated_scan, x, gate, h0, lengths)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, lengths):
        h, last, states = _native.gated_scan(x, gate, h0, lengths, True)
        ctx.save_for_backward(x, gate, states, lengths)
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def backward(ctx, dh, dlast):
        if torch.is_grad_enabled():
            raise RuntimeError("gated_scan can be differentiated once only (create_graph=True)")
        if dh is None and dlast is None:
            return None, None, None, None
        x, gate, states, lengths = ctx.saved_tensors
        return (*_native.gated_scan_backward(x, gate, lengths, states, dh, dlast,
                                             ctx.needs_input_grad[2]), None)


def gated_scan_step(x, gate, state, slots=None):
    """One sample of each of B streams: x and gate [B, D] (or gate None and x
    [B, 2 D], as for gated_scan), state [rows, D] float32, updated in place.
    slots [B] (int32 or int64) gives each stream's row of state (None: row b);
    a slot outside [0, rows), such as -1, marks a stream without a sample now:
    no state changes and its output is 0.  Slots in use must differ.

    Returns h [B, D] of x's type, the streams' new states.  No gradient."""
    slots = _int32(slots, "slots", state.shape[0])
    if torch.is_grad_enabled() and (x.requires_grad or state.requires_grad
                                    or (gate is not None and gate.requires_grad)):
        raise RuntimeError("gated_scan_step has no gradient (its state is updated in place); "
                           "call it under torch.no_grad(), or use gated_scan")
    ext = _ext.module()
    if ext is None:
        return _native.gated_scan_step(x, gate, state, slots)
    return _ext.call(ext.gated_scan_step, x, gate, state, slots)
