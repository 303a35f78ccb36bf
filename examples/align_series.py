"""Train a network that aligns long 1D signals: it reads a warped, noisy signal
of its own length and predicts the theta of the CPAB warp that aligns it with
the template; then follow one signal sample by sample.

    python examples/align_series.py [--steps 300] [--length 512] [--state-bits 8]
                                    [--projection-bits 8] [--muon]

Every sequence operator of the package works here as in use: rms_norm and
gated_scan (with ragged lengths) in the network and its gradient, with its
projections' products in 8 bits if asked for; AdamW with 32- or 8-bit states,
or Muon for the blocks' matrices beside it; gated_scan_step,
rms_norm_quantized and matmul_quantized in the stream.
"""
import argparse
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "fg-cpab_b200"))

import torch  # noqa: E402

from cpab.optim import AdamW, Muon  # noqa: E402
from cpab.pytorch.localizer import SeriesLocalizer  # noqa: E402
from cpab.pytorch.warp import CpabWarp  # noqa: E402


def template(length, device):
    t = torch.linspace(0, 1, length, device=device)
    return (torch.sin(12 * t) * torch.exp(-2 * t) + (t > 0.6) * (t - 0.6))[None, None]


def batch(warp, base, size, noise, g):
    """Warped noisy copies of the template, and the thetas that made them."""
    theta = 0.5 * torch.randn(size, warp.theta_dim, generator=g, device=base.device)
    with torch.no_grad():
        x = warp(base.expand(size, -1, -1), theta)
    return x + noise * torch.randn(x.shape, generator=g, device=x.device), theta


def with_time(x):
    """The signal and when its samples come, as the network's two channels."""
    t = torch.linspace(-1, 1, x.shape[2], device=x.device).expand(x.shape[0], 1, -1)
    return torch.cat([x, t], 1)


def train(steps=300, length=512, size=32, state_bits=32, width=128, depth=2, lr=8e-3, seed=0,
          device="cuda", report=50, tess=8, projection_bits=16, muon=False):
    """Returns (network, warp, losses)."""
    torch.manual_seed(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    warp = CpabWarp([tess], padding_mode="border").to(device)
    net = SeriesLocalizer(2, warp.theta_dim, width, depth, projection_bits=projection_bits).to(device)
    matrices = [p for p in net.blocks.parameters() if p.dim() == 2] if muon else []
    opts = [AdamW([p for p in net.parameters() if not any(p is q for q in matrices)], lr=lr,
                  betas=(0.9, 0.98), weight_decay=0.01, state_bits=state_bits)]
    if muon:
        opts.append(Muon(matrices, lr=lr, weight_decay=0.01, adjust_lr_fn="match_rms_adamw"))
    base = template(length, device)
    losses = []
    for step in range(steps):
        x, _ = batch(warp, base, size, 0.02, g)
        lengths = torch.randint(length // 2, length + 1, (size,), generator=g, device=device)
        lengths[0] = length
        theta = net(with_time(x), lengths)
            # (the warp of -theta undoes that of theta: what the network has to find)
        aligned = warp(x, theta)
        seen = torch.arange(length, device=device)[None, None] < lengths[:, None, None]
        loss = ((aligned - base).square() * seen).sum() / seen.sum()
        net.zero_grad()
        loss.backward()
        for opt in opts:
            opt.step()
        losses.append(loss.detach())
        if report and (step + 1) % report == 0:
            print("step %d: loss %.5f" % (step + 1, torch.stack(losses[-report:]).mean().item()))
    return net, warp, torch.stack(losses).tolist()


def follow(net, x, quantized=False):
    """theta after every sample of one signal x [2, L] (with its times)."""
    states = net.new_states(1)
    return torch.stack([net.step(x[:, t][None], states, quantized=quantized)[0]
                        for t in range(x.shape[1])])


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=300)
    ap.add_argument("--length", type=int, default=512)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    ap.add_argument("--projection-bits", type=int, default=16, choices=(8, 16))
    ap.add_argument("--muon", action="store_true")
    a = ap.parse_args()
    net, warp, losses = train(a.steps, a.length, state_bits=a.state_bits,
                              projection_bits=a.projection_bits, muon=a.muon)
    print("loss: %.5f (first 20 steps), %.5f (last 20)" % (sum(losses[:20]) / 20, sum(losses[-20:]) / 20))
    x, theta = batch(warp, template(a.length, "cuda"), 1, 0.02, torch.Generator("cuda").manual_seed(7))
    x = with_time(x)
    path = follow(net, x[0])
    with torch.no_grad():
        whole = net(x)[0]
    print("theta of the stream after its last sample against the whole signal's: %.2e apart"
          % (path[-1] - whole).abs().max().item())
    low = follow(net.quantize(), x[0], quantized=True)
    print("with 8-bit norms and projections: %.2e apart" % (low[-1] - whole).abs().max().item())


if __name__ == "__main__":
    main()
