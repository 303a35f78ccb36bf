"""The 8-bit projections and Muon together, as a network uses them: a localiser with
projection_bits=8 trained by Muon beside AdamW, then answered sample by sample with
8-bit products.

Codes are off by 2^-4 of a value at most, about 2.5% rms, inputs and weights alike;
a projection of 48 or more such terms by 3.6% of its size.  Two blocks of two
projections, forward and back, are eight of independent sign: 10%, and so is the
angle between the gradients of a network with 8-bit projections and one without:
a cosine of 0.99, 0.95 for any one tensor."""
import importlib.util
import os

import pytest
import torch

from cpab.optim import AdamW, Muon
from cpab.pytorch.localizer import SeriesLocalizer

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def network(bits, width=48):
    torch.manual_seed(0)
    net = SeriesLocalizer(3, 11, width, 2, projection_bits=bits).to(DEV)
    torch.nn.init.normal_(net.head.weight, std=0.3)
    return net


def test_gradients_are_those_of_the_network():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 90, generator=g).to(DEV)
    up = torch.randn(5, 11, generator=g).to(DEV)
    lengths = torch.tensor([90, 1, 0, 33, 64], device=DEV)
    grads, thetas = [], []
    for bits in (16, 8):
        net = network(bits)
        theta = net(x, lengths)
        theta.backward(up)
        thetas.append(theta.detach())
        grads.append({k: p.grad.flatten() for k, p in net.named_parameters()})
    assert not thetas[1][2].any()
    assert (thetas[0] - thetas[1]).norm() <= 0.1 * thetas[0].norm()
    for k in grads[0]:
        assert torch.nn.functional.cosine_similarity(grads[0][k], grads[1][k], dim=0) >= 0.95, k


def test_samples_past_a_series_end_do_not_matter():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 70, generator=g).to(DEV)
    n = torch.tensor([70, 1, 0, 33], device=DEV)
    past = torch.arange(70, device=DEV)[None, None] >= n[:, None, None]
    seen = []
    for fill in (0.0, float("nan"), 3e38):
        net = network(8)
        theta = net(torch.where(past, torch.full_like(x, fill), x), n)
        theta.sum().backward()
        seen.append([theta.detach(), *(p.grad for p in net.parameters())])
    assert all(torch.equal(a, b) for other in seen[1:] for a, b in zip(seen[0], other))


def test_training_and_answering():
    net = network(8, width=64)
    matrices = [p for p in net.blocks.parameters() if p.dim() == 2]
    others = [p for p in net.parameters() if not any(p is q for q in matrices)]
    opts = [Muon(matrices, lr=1e-3, adjust_lr_fn="match_rms_adamw"), AdamW(others, lr=1e-3, state_bits=8)]
    g = torch.Generator().manual_seed(2)
    x, goal = torch.randn(6, 3, 80, generator=g).to(DEV), torch.randn(6, 11, generator=g).to(DEV)
    before = [p.detach().clone() for p in net.parameters()]
    for _ in range(4):
        net.zero_grad()
        (net(x) - goal).square().mean().backward()
        for opt in opts:
            opt.step()
    assert all(p.isfinite().all() and not torch.equal(p, q) for p, q in zip(net.parameters(), before))
    net.quantize()
    states = net.new_states(6)
    for t in range(80):
        theta = net.step(x[:, :, t], states, quantized=True)
    with torch.no_grad():
        whole = net(x)
    assert (theta - whole).norm() <= 0.15 * whole.norm()


def test_example_runs():
    spec = importlib.util.spec_from_file_location("align_series", os.path.join(ROOT, "examples", "align_series.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    net, warp, losses = ex.train(steps=3, length=128, size=8, width=64, report=0, projection_bits=8, muon=True)
    assert len(losses) == 3 and all(loss == loss for loss in losses)
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
