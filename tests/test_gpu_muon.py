"""orthogonalize, muon_ and Muon against their formulas in float64.

Tolerances (relative 2-norm of a matrix).  16-bit types over 256 rows (on the
short side; smaller ones are multiplied as float32 ones): both operands of each
of the three products of a step are rounded to halves (2^-11 at most, each), an
error that later steps multiply as they multiply the values themselves: 5 steps
of 3 products of independent errors, 30 roundings, each sqrt(1/3) of its most in
the mean: sqrt(30 / 3) 2^-11 = 1.6e-3, and up to twice that where the singular
values that a step multiplies most (3.4) carry the errors: 3.2e-3; plus half a
step of the result's type.  float32: operands keep 22 bits (2^-22, the
remainders' product dropped: 2^-22), sums are cut at most 48 times a segment
(48 2^-24): 3.3e-6 a product, 15 of them and twice: 1e-4 at most, in the mean
(sqrt(15) and twice) 2.6e-5."""
import contextlib
import copy
import math

import pytest
import torch

from cpab import _ext
from cpab.optim import COEFFICIENTS, Muon, muon_, orthogonalize

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def most(dtype, shape):
    return 3.2e-3 if dtype != F32 and min(shape[-2:]) > 256 else 2.6e-5


@pytest.fixture(params=["ext", "python"])
def path(request):
    with _ext.python_path() if request.param == "python" else contextlib.nullcontext():
        yield request.param


def exact(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = x @ x.mT
        x = a * x + (b * A + c * A @ A) @ x
    return x.mT if tall else x


def off(got, want):
    return ((got.double() - want).norm() / want.norm().clamp_min(1e-300)).item()


def matrices(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = min(4, m, n)
    low = torch.randn(*shape[:-1], r, generator=g) @ torch.randn(*shape[:-2], r, n, generator=g)
    return ((torch.randn(shape, generator=g) + 0.5 * low) * scale).to(DEV, dtype)


SHAPES = [(1, 1), (1, 7), (5, 1), (3, 17), (16, 16), (49, 130), (130, 3), (128, 128), (130, 260), (260, 130),
          (3, 130, 260), (193, 200), (257, 300), (640, 256), (2, 3, 65, 40), (500, 1000), (1000, 1003), (40, 3000),
          (129, 4097), (3, 150, 2000), (3000, 300)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype, path):
    x = matrices(shape, dtype)
    y = orthogonalize(x)
    assert y.dtype == dtype and y.shape == x.shape
    want = exact(x)
    for got, w in zip(y.reshape(-1, *shape[-2:]), want.reshape(-1, *shape[-2:])):
        assert off(got, w) <= most(dtype, shape) + STEP[dtype]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2048, 1500), (1300, 4100), (6, 700, 900)])
def test_large_ones(shape, dtype, path):
    x = matrices(shape, dtype, 1, 1e-4)
    assert off(orthogonalize(x), exact(x)) <= most(dtype, shape) + STEP[dtype]


@pytest.mark.parametrize("shape", [(64, 64), (130, 260), (300, 500)])
def test_small_directions_beside_strong_ones(shape):
    """Eight directions a hundred times the others: halves alone would lose the
    rest (4e-2 off); the remainders in a X keep them."""
    g = torch.Generator().manual_seed(3)
    x = (0.01 * torch.randn(shape, generator=g) +
         torch.randn(shape[0], 8, generator=g) @ torch.randn(8, shape[1], generator=g)).to(DEV)
    assert off(orthogonalize(x), exact(x)) <= most(F32, (1, 1))
    assert off(orthogonalize(x.to(BF16)), exact(x.to(BF16))) <= most(BF16, shape) + STEP[BF16]


def test_singular_values_come_near_1():
    x = matrices((96, 160), F32)
    y = orthogonalize(x)
    s = torch.linalg.svdvals(y.double())
    assert 0.6 < s.min() and s.max() < 1.3
    u, _, v = torch.linalg.svd(x.double(), full_matrices=False)
    d = u.T @ y.double() @ v.T
    assert (d - torch.diag(d.diagonal())).abs().max() < 1e-4


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e25, 3e37])
def test_any_size_of_values(scale, path):
    """The norm is summed in float64; eps counts beside norms near it."""
    x = matrices((40, 70), F32, 2) * scale
    assert x.isfinite().all()
    want = exact(x)
    assert off(orthogonalize(x), want) <= most(F32, (1, 1))


def test_zeros_nan_and_empty(path):
    z = torch.zeros(2, 30, 40, device=DEV)
    assert not orthogonalize(z).any()
    for bad in (float("nan"), float("inf")):
        x = matrices((3, 150, 300), F32)
        x[1, 7, 9] = bad
        y = orthogonalize(x)
        assert y[1].isnan().all() and not y[0].isnan().any() and not y[2].isnan().any()
        assert off(y[0], exact(x[0])) <= most(F32, (1, 1))
    for shape in ((0, 5, 6), (3, 0, 6), (4, 0)):
        assert orthogonalize(torch.empty(shape, device=DEV)).shape == shape


def test_other_steps_coefficients_and_strides(path):
    x = matrices((90, 120), F32)
    for steps, coefficients in ((1, COEFFICIENTS), (2, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375))):
        assert off(orthogonalize(x, steps, coefficients), exact(x, steps, coefficients)) <= 2 * most(F32, (1, 1)) * max(1, steps / 5)
    for v in (x.t(), x[::2], x[:, 3:77], x[:1].expand(4, -1)):
        assert off(orthogonalize(v), exact(v)) <= most(F32, (1, 1))
    assert torch.equal(orthogonalize(x, eps=1e-3), orthogonalize(x.clone(), eps=1e-3))


@pytest.mark.parametrize("shape", [(130, 260), (700, 900)])
def test_streams_graphs_and_runs(shape, path):
    x = matrices(shape, F32)
    want = orthogonalize(x)
    assert torch.equal(orthogonalize(x), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize(x)
    side.synchronize()
    assert torch.equal(got, want)
    a, b = x.clone(), x.clone()
    graphs, outs = [], []
    for t in (a, b):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(orthogonalize(t))
    b.copy_(matrices(shape, F32, 9))
    other = orthogonalize(b)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], other)


# ---- the step --------------------------------------------------------------------

def step64(p, g, m, lr, momentum, nesterov, decay, adjust, **kw):
    p, g, m = p.double(), g.double(), m.double()
    m = momentum * m + (1 - momentum) * g
    o = exact((1 - momentum) * g + momentum * m if nesterov else m, **kw)
    r = math.sqrt(max(1, p.shape[0] / p.shape[1])) if adjust == "original" else 0.2 * math.sqrt(max(p.shape))
    return p * (1 - lr * decay) - lr * r * o, m, lr * r * o


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("adjust,nesterov", [("original", True), ("match_rms_adamw", True), ("original", False)])
def test_step(dtype, adjust, nesterov, path):
    """Matrices of several shapes, some alike, tall and wide; one of a network's width."""
    shapes = [(130, 3), (260, 130), (130, 130), (260, 130), (49, 130), (1, 9), (300, 700), (700, 300), (64, 64)]
    ps = [matrices(s, dtype, k, 0.05) for k, s in enumerate(shapes)]
    gs = [matrices(s, dtype, 50 + k, 10.0 ** -(k % 3)) for k, s in enumerate(shapes)]
    ms = [matrices(s, F32, 90 + k, 10.0 ** -(k % 3)) for k, s in enumerate(shapes)]
    lr, momentum, decay = 0.02, 0.9, 0.3
    want = [step64(p, g, m, lr, momentum, nesterov, decay, adjust) for p, g, m in zip(ps, gs, ms)]
    keep = [g.clone() for g in gs]
    versions = [p._version for p in ps]
    muon_(ps, gs, ms, lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=decay, adjust_lr=adjust)
    for p, m, (wp, wm, move) in zip(ps, ms, want):
        # two products and their sum, rounded to float32
        assert ((m.double() - wm).abs() <= 4 * 2.0 ** -24 * (wm.abs() + 2 * wm.abs().max())).all()
        assert (p.double() - wp).norm() <= most(dtype, p.shape) * move.norm() + (STEP[dtype] + 2.0 ** -22) * (wp.norm() + move.norm())
    assert all(torch.equal(a, b) for a, b in zip(gs, keep))
    assert all(p._version > v for p, v in zip(ps, versions))


def test_many_matrices(path):
    """More than one launch's: 200 small ones of 11 shapes."""
    ps = [matrices((8 + k % 11, 20), F32, k) for k in range(200)]
    gs = [matrices((8 + k % 11, 20), F32, 300 + k) for k in range(200)]
    ms = [torch.zeros_like(p) for p in ps]
    want = [step64(p, g, m, 0.1, 0.9, True, 0.0, "original") for p, g, m in zip(ps, gs, ms)]
    muon_(ps, gs, ms, lr=0.1, momentum=0.9, weight_decay=0.0)
    for p, (wp, _, move) in zip(ps, want):
        assert (p.double() - wp).norm() <= most(F32, (1, 1)) * move.norm() + 2.0 ** -22 * (wp.norm() + move.norm())


def test_many_larger_matrices_of_mixed_types(path):
    """More shapes and matrices than a sequence of launches takes, float32 and 16-bit
    ones, matrices of none, small ones among them."""
    kinds = [((130 + 7 * (k % 10), 150), F32) for k in range(140)] + [((300, 260 + 8 * k), BF16) for k in range(3)] + \
        [((0, 5), F32), ((20, 30), BF16), ((12, 200), F16), ((280, 280), F16)]
    ps = [matrices(s, t, k, 0.05) if 0 not in s else torch.empty(s, device=DEV) for k, (s, t) in enumerate(kinds)]
    gs = [matrices(s, t, 300 + k) if 0 not in s else torch.empty(s, device=DEV) for k, (s, t) in enumerate(kinds)]
    ms = [torch.zeros(s, device=DEV) for s, _ in kinds]
    want = [step64(p, g, m, 0.1, 0.9, True, 0.1, "original") if p.numel() else None for p, g, m in zip(ps, gs, ms)]
    muon_(ps, gs, ms, lr=0.1, momentum=0.9, weight_decay=0.1)
    for p, w in zip(ps, want):
        if w is not None:
            wp, _, move = w
            assert (p.double() - wp).norm() <= most(p.dtype, p.shape) * move.norm() + \
                (STEP[p.dtype] + 2.0 ** -22) * (wp.norm() + move.norm())


@pytest.mark.parametrize("shape", [(70, 130, 140), (3000, 8, 9), (1, 70000)])
def test_many_in_a_batch(shape, path):
    x = matrices(shape, F32, 4)
    y, want = orthogonalize(x), exact(x)
    off_ = (y.double() - want).flatten(-2).norm(dim=-1) / want.flatten(-2).norm(dim=-1)
    assert off_.max() <= most(F32, shape)


def test_learning_rate_on_the_device_for_all_kinds(path):
    shapes = [(300, 400), (400, 300), (20, 30)]
    a = [matrices(s, F32, k, 0.05) for k, s in enumerate(shapes)]
    b = [p.clone() for p in a]
    gs = [matrices(s, F32, 9 + k) for k, s in enumerate(shapes)]
    for ps, lr in ((a, torch.tensor(0.25, device=DEV)), (b, 0.25)):
        muon_(ps, gs, [torch.zeros_like(p) for p in ps], lr=lr)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def net(dtype=F32, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 40, bias=False), torch.nn.Linear(40, 40, bias=False),
                               torch.nn.Linear(40, 7, bias=False)).to(DEV, dtype)


def fill(model, seed):
    for k, p in enumerate(model.parameters()):
        p.grad = matrices(tuple(p.shape), p.dtype, seed + k)


def test_optimizer(path):
    model, opt = net(), None
    opt = Muon([{"params": [model[0].weight]}, {"params": [model[1].weight, model[2].weight], "lr": 0.05}], lr=0.01)
    ps = [p.detach().double() for p in model.parameters()]
    ms = [torch.zeros_like(p) for p in ps]
    for step in range(3):
        fill(model, 10 * step)
        model[2].weight.grad = None if step == 1 else model[2].weight.grad
        for k, p in enumerate(model.parameters()):
            if p.grad is not None:
                ps[k], ms[k], _ = step64(ps[k], p.grad, ms[k], 0.01 if k == 0 else 0.05, 0.95, True, 0.1, "original")
        opt.step()
    for p, want, m in zip(model.parameters(), ps, ms):
        assert off(p.detach(), want) <= 1e-5 and off(opt.state[p]["momentum_buffer"], m) <= 1e-6
    assert opt.step(lambda: torch.ones(())) == 1


def test_state_dicts_and_copies(path):
    a = net()
    opt = Muon(a.parameters(), lr=0.02, weight_decay=0.01)
    fill(a, 0)
    opt.step()
    b = net()
    b.load_state_dict(a.state_dict())
    other = Muon(b.parameters(), lr=0.5)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for o, n in ((opt, a), (other, b)):
        fill(n, 5)
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    # torch's own state dict, whose momenta are of the parameters' type
    c = net(BF16)
    theirs = torch.optim.Muon(c.parameters(), lr=0.02)
    fill(c, 0)
    theirs.step()
    mine = Muon(c.parameters())
    mine.load_state_dict(theirs.state_dict())
    assert mine.param_groups[0]["lr"] == 0.02
    assert all(mine.state[p]["momentum_buffer"].dtype == F32 for p in c.parameters())
    fill(c, 3)
    mine.step()
    assert all(p.isfinite().all() for p in c.parameters())
    copy.deepcopy(mine).step()


def test_captured_step_follows_a_learning_rate_on_the_device(path):
    a, b = net(), net()
    lr = torch.tensor(0.01, device=DEV)
    oa, ob = Muon(a.parameters(), lr=lr), Muon(b.parameters(), lr=0.01)
    for n, o in ((a, oa), (b, ob)):
        fill(n, 0)
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for rate in (0.01, 0.2):
        lr.fill_(rate)
        for group in ob.param_groups:
            group["lr"] = float(lr)
        graph.replay()
        ob.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    fresh = net()
    fill(fresh, 0)
    opt = Muon(fresh.parameters())
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()


def test_refusals(path):
    p, g, m = (torch.zeros(4, 6, device=DEV) for _ in range(3))
    for bad in (dict(params=[p.to(BF16)]), dict(momenta=[m.to(BF16)])):
        with pytest.raises(TypeError):
            muon_(**{**dict(params=[p], grads=[g], momenta=[m]), **bad}, lr=0.1)
    for bad in (dict(grads=[g[:3]]), dict(params=[p.t()], grads=[g.t()], momenta=[m.t()]), dict(grads=[]),
                dict(params=[p[0]], grads=[g[0]], momenta=[m[0]])):
        with pytest.raises(ValueError):
            muon_(**{**dict(params=[p], grads=[g], momenta=[m]), **bad}, lr=0.1)
    with pytest.raises(RuntimeError, match="twice"):
        muon_([p, p], [g, g], [m, m.clone()], lr=0.1)
    with pytest.raises(RuntimeError, match="device"):
        muon_([p], [g.cpu()], [m], lr=0.1)
    with pytest.raises(ValueError, match="lr"):
        muon_([p], [g], [m], lr=torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError, match="outgrow"):
        orthogonalize(p, coefficients=(100.0, -4.0, 2.0))
    with pytest.raises(RuntimeError, match="steps"):
        orthogonalize(p, steps=0)
    with pytest.raises(RuntimeError, match="no gradient"):
        orthogonalize(p.clone().requires_grad_(True))
    with pytest.raises(TypeError):
        orthogonalize(p.double())
    with pytest.raises(ValueError):
        orthogonalize(p[0])
    muon_([], [], [], lr=0.1)
