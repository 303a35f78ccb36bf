"""A localisation network for long signals: predicts theta of a CPAB warp from
series of samples, with the sequence operators of this package.

    series [B, channels, L] -> samples' embedding -> depth blocks of
        y, s = rms_norm(update, weight, residual=s)
        h, _ = gated_scan(in_proj(y))          # inputs and gates in one projection
        update = out_proj(h)
    -> rms_norm at each series' last sample -> head -> theta [B, theta_dim]

The same weights answer sample by sample (step): the recurrence's states are
all that is kept of a stream, so theta follows a signal as it arrives.  No
counterpart in the reference, whose localisation networks read images.
"""
import torch
import torch.nn as nn

from .norm import rms_norm, rms_norm_quantized
from .projection import linear_quantized, matmul_quantized
from .recurrence import gated_scan, gated_scan_step


class RecurrentBlock(nn.Module):
    def __init__(self, width):
        super().__init__()
        self.norm = nn.Parameter(torch.ones(width))
        self.in_proj = nn.Linear(width, 2 * width)
        self.out_proj = nn.Linear(width, width)
        with torch.no_grad():
            # gates of 0.73 to 0.999: memories of a few to a thousand samples
            self.in_proj.bias[width:] = torch.linspace(1.0, 7.0, width)
            self.out_proj.weight.mul_(0.5)


class SeriesLocalizer(nn.Module):
    """SeriesLocalizer(channels, theta_dim, width, depth)(series, lengths) ->
    theta; theta starts at 0 (the identity warp).  projection_bits=8: the blocks'
    projections and their gradients are 8-bit products (linear_quantized).  A training
    step on 32 series of 512 samples, 16 and 8 bits (us): width 128 in bfloat16 987 and
    899, 2048 2442 and 2105; in float32, whose library products take no tensor cores
    unless told to, 1001 and 889, 42004 and 2753."""

    def __init__(self, channels, theta_dim, width=128, depth=2, eps=1e-6, projection_bits=16):
        super().__init__()
        if depth < 1 or width < 1:
            raise ValueError("width and depth must be at least 1")
        if projection_bits not in (8, 16):
            raise ValueError("projection_bits must be 8 or 16, got %r" % (projection_bits,))
        self.projection_bits = projection_bits
        self.channels, self.theta_dim, self.width, self.eps = channels, theta_dim, width, eps
        self.embed = nn.Linear(channels, width)
        self.blocks = nn.ModuleList(RecurrentBlock(width) for _ in range(depth))
        self.norm = nn.Parameter(torch.ones(width))
        self.head = nn.Linear(width, theta_dim)
        nn.init.zeros_(self.head.weight)
        nn.init.zeros_(self.head.bias)

    def forward(self, series, lengths=None):
        """series [B, channels, L], lengths [B] or None (all L) -> theta
        [B, theta_dim] from each series' first lengths[b] samples (0 for a
        series without one: the identity).  What series holds after them does
        not matter, nor to the gradients."""
        if series.dim() != 3 or series.shape[1] != self.channels or series.shape[2] < 1:
            raise ValueError("series must be [B, %d, L], got %s" % (self.channels, tuple(series.shape)))
        if lengths is not None:
            # (gated_scan passes over them by itself, but the weights' gradients of
            # the norms and projections would be sums with 0 x NaN)
            seen = torch.arange(series.shape[2], device=series.device) < lengths[:, None, None]
            series = series.masked_fill(~seen, 0.0)
        s = self.embed(series.transpose(1, 2))
        update = None
        for block in self.blocks:
            if update is None:
                y = rms_norm(s, block.norm, eps=self.eps)
            else:
                y, s = rms_norm(update, block.norm, residual=s, eps=self.eps)
            h, _ = gated_scan(self._project(block.in_proj, y), lengths=lengths)
            update = self._project(block.out_proj, h)
        if lengths is None:
            return self._theta(update[:, -1], s[:, -1])
        at = (lengths.long().clamp(1, series.shape[2]) - 1)[:, None, None].expand(-1, 1, self.width)
        theta = self._theta(update.gather(1, at)[:, 0], s.gather(1, at)[:, 0])
        return theta * (lengths > 0)[:, None]

    def _project(self, proj, x):
        if self.projection_bits == 8:
            return linear_quantized(x, proj.weight, proj.bias)
        return proj(x)

    def _theta(self, update, s):
        y, _ = rms_norm(update.contiguous(), self.norm, residual=s.contiguous(), eps=self.eps)
        return self.head(y).float()

    def new_states(self, rows, device=None):
        """States of `rows` streams that have had no sample: [depth, rows, width]."""
        return torch.zeros(len(self.blocks), rows, self.width, dtype=torch.float32,
                           device=device if device is not None else self.norm.device)

    def quantize(self):
        """Keep the blocks' input projections in 8 bits too (e4m3 codes, a scale
        per output), for step(..., quantized=True).  Call again after training."""
        if self.width % 16:
            raise ValueError("8-bit projections need a width that is a multiple of 16")
        for block in self.blocks:
            w = block.in_proj.weight.detach().float()
            scale = (w.abs().amax(1) / 448.0).clamp_min(2.0 ** -126)
            block.in_proj_q = (w / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
            block.in_proj_scale = scale
        return self

    @torch.no_grad()
    def step(self, samples, states, slots=None, quantized=False):
        """One sample of each of B streams: samples [B, channels], states from
        new_states, updated in place, slots [B] the streams' rows of it (None:
        row b; -1: no sample now, whose theta means nothing).  Returns theta
        [B, theta_dim] of the streams so far, as forward gives for them (with
        projection_bits=8 the projections are its 8-bit ones, whose weights are
        quantized at every step).  quantized, whatever projection_bits is: norms
        and input projections in 8 bits with the weights that quantize keeps,
        whose products are rounded to 16 bits; output projections in the
        weights' type."""
        s = self.embed(samples)
        update = None
        for k, block in enumerate(self.blocks):
            if quantized:
                out = rms_norm_quantized(s if update is None else update, block.norm,
                                         residual=None if update is None else s, eps=self.eps)
                if update is not None:
                    s = out[2]
                z = matmul_quantized(out[0], out[1], block.in_proj_q, block.in_proj_scale)
                z = z.to(s.dtype) + block.in_proj.bias
            else:
                if update is None:
                    y = rms_norm(s, block.norm, eps=self.eps)
                else:
                    y, s = rms_norm(update, block.norm, residual=s, eps=self.eps)
                z = self._project(block.in_proj, y)
            h = gated_scan_step(z, None, states[k], slots)
            update = block.out_proj(h) if quantized else self._project(block.out_proj, h)
        return self._theta(update, s)
