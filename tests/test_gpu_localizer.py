"""The localisation network of cpab.pytorch.localizer against the same network
in plain float64 torch, and the example that trains it.

Tolerances: the operators' own are 1e-6 to 5e-6 of a float32 tensor; the
projections between them are torch's float32 products, a sum of `width` terms
(1e-6); two blocks, forward and back, are below 30 such steps: 1e-4.  A 16-bit
network rounds each of them to 2^-8: 30 roundings of independent sign, 5%."""
import importlib.util
import os

import pytest
import torch

from cpab.pytorch.localizer import SeriesLocalizer

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def network(channels=3, theta=11, width=48, depth=2, seed=0):
    torch.manual_seed(seed)
    net = SeriesLocalizer(channels, theta, width, depth).to(DEV)
    torch.nn.init.normal_(net.head.weight, std=0.3)
    return net


def plain(net, series, lengths):
    """The network in float64, sample by sample; parameters as given."""
    def norm(v, w):
        return v / (v.square().mean(-1, keepdim=True) + net.eps).sqrt() * w
    P = {k: v.detach().double().requires_grad_(True) for k, v in net.named_parameters()}
    s = series.double().transpose(1, 2) @ P["embed.weight"].t() + P["embed.bias"]
    B, L, W = s.shape
    n = torch.full((B,), L, device=s.device) if lengths is None else lengths.long().clamp(0, L)
    update = torch.zeros_like(s)
    for k in range(len(net.blocks)):
        p = lambda name: P["blocks.%d.%s" % (k, name)]  # noqa: E731
        s = s + update
        z = norm(s, p("norm")) @ p("in_proj.weight").t() + p("in_proj.bias")
        a, h, hs = torch.sigmoid(z[..., W:]), torch.zeros(B, W, device=s.device, dtype=s.dtype), []
        for t in range(L):
            h = a[:, t] * h + (1 - a[:, t]) * z[:, t, :W]
            hs.append(h)
        h = torch.stack(hs, 1) * (torch.arange(L, device=s.device)[None] < n[:, None])[..., None]
        update = h @ p("out_proj.weight").t() + p("out_proj.bias")
    at = (n.clamp_min(1) - 1)
    last = (s + update)[torch.arange(B, device=s.device), at]
    theta = norm(last, P["norm"]) @ P["head.weight"].t() + P["head.bias"]
    return theta * (n > 0)[:, None], P


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("width", [48, 33])
def test_network_and_gradient(ragged, width):
    net = network(width=width)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 70, generator=g).to(DEV)
    n = torch.tensor([70, 1, 0, 33], device=DEV) if ragged else None
    theta = net(x, n)
    ref, P = plain(net, x, n)
    assert theta.shape == (4, 11) and (theta - ref).norm() <= 1e-4 * ref.norm()
    up = torch.randn(4, 11, generator=g).to(DEV)
    theta.backward(up)
    ref.backward(up.double())
    for k, v in net.named_parameters():
        assert (v.grad - P[k].grad).norm() <= 1e-4 * P[k].grad.norm().clamp_min(1e-6), k
    if ragged:
        assert not theta[2].any()


def test_network_in_16_bits():
    net = network().bfloat16()
    x = torch.randn(4, 3, 70, generator=torch.Generator().manual_seed(1)).to(DEV)
    theta = net(x.bfloat16())
    ref, _ = plain(net, x.bfloat16(), None)
    assert (theta - ref).norm() <= 0.05 * ref.norm()


def test_stream_follows_the_series():
    net = network()
    x = torch.randn(3, 3, 40, generator=torch.Generator().manual_seed(2)).to(DEV)
    states = net.new_states(5)
    slots = torch.tensor([4, 0, 2], device=DEV)
    for t in range(40):
        # stream 1 has samples at even times only
        at = slots.clone()
        if t % 2:
            at[1] = -1
        theta = net.step(x[:, :, t], states, at)
        if t in (0, 7, 39):
            with torch.no_grad():
                want = net(x[:, :, :t + 1])
            assert (theta[[0, 2]] - want[[0, 2]]).abs().max() <= 1e-4 * want.abs().max()
    with torch.no_grad():
        want = net(x[1:2, :, ::2])
    got = net.step(x[1:2, :, 0], net.new_states(1))
    again = net.new_states(1)
    for t in range(0, 40, 2):
        got = net.step(x[1:2, :, t], again)
    assert (got - want).abs().max() <= 1e-4 * want.abs().max()
    assert torch.allclose(again[:, 0], states[:, 0], atol=1e-5) and not states[:, 1].any()


def test_8_bit_stream():
    """Codes are off by 2^-4 of a value at most (about 2.5% rms), weights and
    inputs alike; a product of 48 such terms by 3.6% of its size; two blocks."""
    net = network(width=48).quantize()
    x = torch.randn(2, 3, 30, generator=torch.Generator().manual_seed(3)).to(DEV)
    a, b = net.new_states(2), net.new_states(2)
    for t in range(30):
        full = net.step(x[:, :, t], a)
        low = net.step(x[:, :, t], b, quantized=True)
    assert (full - low).norm() <= 0.15 * full.norm()
    with pytest.raises(ValueError, match="16"):
        network(width=33).quantize()
    with pytest.raises(ValueError, match="series"):
        net(x[:, :2])


@pytest.mark.parametrize("bits", [32, 8])
def test_example_learns(bits):
    """The example's loss falls: to less than half within 120 steps."""
    spec = importlib.util.spec_from_file_location("align_series", os.path.join(ROOT, "examples", "align_series.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    net, warp, losses = ex.train(steps=120, length=192, size=16, state_bits=bits, width=64, report=0)
    first, last = sum(losses[:10]) / 10, sum(losses[-10:]) / 10
    assert last < 0.5 * first, (first, last)
    x, _ = ex.batch(warp, ex.template(192, DEV), 1, 0.02, torch.Generator(DEV).manual_seed(7))
    x = ex.with_time(x)
    with torch.no_grad():
        whole = net(x)[0]
    path = ex.follow(net, x[0])
    assert path.shape == (192, warp.theta_dim)
    assert (path[-1] - whole).abs().max() <= 1e-3 * whole.abs().max().clamp_min(1.0)


def test_samples_past_a_series_end_do_not_matter():
    """Whatever they hold: theta and the gradients are those of zeros there."""
    net = network()
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 70, generator=g).to(DEV)
    up = torch.randn(4, 11, generator=g).to(DEV)
    n = torch.tensor([70, 1, 0, 33], device=DEV)
    past = torch.arange(70, device=DEV)[None, None] >= n[:, None, None]
    seen = []
    for fill in (0.0, float("nan"), float("inf"), 3e38):
        net.zero_grad()
        series = torch.where(past, torch.full_like(x, fill), x).requires_grad_(True)
        theta = net(series, n)
        theta.backward(up)
        assert not theta[2].any() and not series.grad[past.expand_as(x)].any()
        seen.append([theta.detach(), series.grad, *(p.grad.clone() for p in net.parameters())])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))
