"""adamw_ and cpab.optim.AdamW against the step's formulas.

The states' arithmetic is elementary float32 operations in a stated order, so
float32 states and 8-bit codes are compared with the same operations on the
CPU bit for bit.  A parameter is compared in float64: three roundings of its
own size (2^-24 each) and a dozen of its update's (1e-6 of it)."""
import contextlib
import copy
import math

import numpy as np
import pytest
import torch

from cpab import _ext, _native
from cpab.optim import AdamW, _step, adamw_
from cpab.pytorch.norm import rms_norm

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16, F8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # unit roundoffs: 11 and 8 significand bits


def hash32(x):
    """PCG-RXS-M-XS on uint32 arrays."""
    x = (x * np.uint32(747796405) + np.uint32(2891336453)).astype(np.uint32)
    x = (((x >> ((x >> np.uint32(28)) + np.uint32(4))) ^ x) * np.uint32(277803737)).astype(np.uint32)
    return (x >> np.uint32(22)) ^ x


def e4m3_values():
    return torch.arange(127, dtype=torch.uint8).view(F8).float().numpy()     # 0 .. 448, ascending


def stochastic(z, u):
    """The code below or above z, above where u / 2^16 exceeds what is left to it."""
    grid = e4m3_values().astype(np.float64)
    k = np.searchsorted(grid, z.astype(np.float64), side="right") - 1
    top = np.minimum(k + 1, len(grid) - 1)
    gap = np.where(k < len(grid) - 1, grid[top] - grid[k], 1.0)
    up = (z - grid[k]) / gap + u / 65536.0 >= 1.0
    return np.where(up, grid[top], grid[k]).astype(np.float32)


def blocks(a):
    n = -(-a.size // 256) * 256
    return np.pad(a, (0, n - a.size)).reshape(-1, 256)


def reference(p, g, m, v, step, scales, lr, betas, eps, wd, seed, index):
    """One tensor's step; numpy float32 states (or codes), float64 parameter."""
    f = np.float32
    b1, b2 = betas
    g32 = g.float().cpu().numpy().ravel()
    if scales is not None:
        sc = scales.cpu().numpy()
        m0 = (blocks(m.float().cpu().numpy().ravel()) * sc[:, :1]).ravel()[:g32.size]
        r0 = (blocks(v.float().cpu().numpy().ravel()) * sc[:, 1:]).ravel()[:g32.size]
        v0 = r0 * r0
    else:
        m0, v0 = m.cpu().numpy().ravel(), v.cpu().numpy().ravel()
    m1 = m0 * f(b1) + g32 * f(1 - b1)
    v1 = v0 * f(b2) + (g32 * g32) * f(1 - b2)
    r1 = np.sqrt(v1)
    t = float(step) + 1
    upd = (m1.astype(np.float64) / (1 - b1 ** t)) / (np.sqrt(v1.astype(np.float64) / (1 - b2 ** t)) + eps)
    p1 = p.double().cpu().numpy().ravel() * (1 - lr * wd) - lr * upd
    if scales is None:
        return p1, lr * upd, m1, v1, None
    ms = np.maximum(np.abs(blocks(m1)).max(1) * (f(1) / f(448)), f(2.0 ** -126))
    rs = np.maximum(blocks(r1).max(1) * (f(1) / f(448)), f(2.0 ** -126))
    with np.errstate(over="ignore"):
        key = hash32(np.array([seed], np.uint32) + np.uint32(index) * np.uint32(0x9E3779B9)
                     + np.uint32(int(t)) * np.uint32(0x85EBCA6B))[0]
        u = hash32(np.arange(g32.size, dtype=np.uint32) + key)
    mq = stochastic((np.abs(blocks(m1)) / ms[:, None]).ravel()[:g32.size], u & np.uint32(0xFFFF))
    rq = stochastic((blocks(r1) / rs[:, None]).ravel()[:g32.size], u >> np.uint32(16))
    rq = np.where((r1 > 0) & (rq == 0), f(2.0 ** -9), rq)
    return p1, lr * upd, np.copysign(mq, m1), rq, np.stack([ms, rs], 1)


def make(sizes, dtype, bits, seed=0, shift=0):
    """Lists of one network's tensors; with `shift` elements before each (odd
    addresses)."""
    g = torch.Generator().manual_seed(seed)

    def at(a, kind):
        buf = torch.empty(a.numel() + shift, device=DEV, dtype=kind)
        buf[shift:] = a.to(DEV).to(kind)
        return buf[shift:]
    L = {k: [] for k in ("p", "g", "m", "v", "step", "scales")}
    for i, n in enumerate(sizes):
        big = 10.0 ** (-2 + i % 3)
        L["p"].append(at(torch.randn(n, generator=g) * 0.1, dtype))
        grad = torch.randn(n, generator=g) * big
        grad[::7] = 0
        L["g"].append(at(grad, dtype))
        m, r = torch.randn(n, generator=g) * 0.3 * big, torch.randn(n, generator=g).abs() * big
        m[::5], r[::5] = 0, 0
        L["step"].append(torch.tensor(float(i * 3), device=DEV))
        if bits == 8:
            nb = -(-n // 256)
            sc = torch.rand(nb, 2, generator=g) * big / 200 + 1e-9
            e = torch.arange(n) // 256
            L["m"].append(at((m / sc[e, 0]).clamp(-448, 448), F8))
            L["v"].append(at((r / sc[e, 1]).clamp(0, 448), F8))
            L["scales"].append(sc.to(DEV))
        else:
            L["m"].append(at(m, F32))
            L["v"].append(at(r * r, F32))
            L["scales"].append(None)
    return L


def copies(L):
    return {k: [None if t is None else t.clone() for t in v] for k, v in L.items()}


HYPER = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def check(L, old, dtype, seed, hyper=HYPER, index=None):
    for i in range(len(L["p"])):
        p1, upd, m1, v1, sc = reference(old["p"][i], L["g"][i], old["m"][i], old["v"][i], old["step"][i],
                                        old["scales"][i], hyper["lr"], hyper["betas"], hyper["eps"],
                                        hyper["weight_decay"], seed, i if index is None else index[i])
        got = L["p"][i].double().cpu().numpy().ravel()
        room = 3 * 2.0 ** -24 * np.abs(p1) + 1e-6 * np.abs(upd) + ROUND[dtype] * np.abs(p1) + \
            (2.0 ** -25 if dtype == F16 else 0)
        assert (np.abs(got - p1) <= room).all(), i
        assert np.array_equal(L["m"][i].float().cpu().numpy().ravel(), m1), i
        assert np.array_equal(L["v"][i].float().cpu().numpy().ravel(), v1), i
        if sc is not None:
            assert np.array_equal(L["scales"][i].cpu().numpy(), sc), i
        assert float(L["step"][i]) == float(old["step"][i]) + 1


SIZES = [1, 3, 255, 256, 257, 2047, 2048, 2049, 10000, 70001]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [0, 1])
def test_step_of_many_tensors(dtype, bits, shift):
    L = make(SIZES, dtype, bits, shift=shift)
    for k in range(2):
        old = copies(L)
        adamw_(L["p"], L["g"], L["m"], L["v"], L["step"], scales=L["scales"] if bits == 8 else None,
               seed=11, **HYPER)
        check(L, old, dtype, 11)


def test_more_tensors_than_a_launch_takes():
    sizes = [1 + (37 * i) % 500 for i in range(600)]
    sizes[5] = 0
    L = make(sizes, F32, 8)
    old = copies(L)
    ws = torch.zeros(1, device=DEV, dtype=torch.int32)
    adamw_(L["p"], L["g"], L["m"], L["v"], L["step"], scales=L["scales"], seed=3, workspace=ws, **HYPER)
    check(L, old, F32, 3)
    assert int(ws) == 0
    adamw_([], [], [], [], [], lr=1e-3)


def test_states_of_both_kinds_in_one_call():
    a, b = make([5000, 300], F32, 8), make([700, 4096], F32, 32, seed=1)
    L = {k: a[k] + b[k] for k in a}
    old = copies(L)
    adamw_(L["p"], L["g"], L["m"], L["v"], L["step"], scales=L["scales"], seed=7, **HYPER)
    check(L, old, F32, 7)


def test_rounding_is_unbiased():
    """The mean of 400 roundings of one value: within 5 standard errors, one
    rounding's deviation being at most half a code's spacing."""
    n = 256
    vals = torch.linspace(1e-3, 1.0, n)
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    total, root = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    for seed in range(400):
        m = torch.zeros(n, device=DEV, dtype=F8)
        v = torch.zeros(n, device=DEV, dtype=F8)
        sc = torch.zeros(1, 2, device=DEV)
        adamw_([p], [vals.to(DEV)], [m], [v], [torch.zeros((), device=DEV)], scales=[sc], seed=seed,
               lr=0.0, betas=(0.5, 0.75))
        total += (m.float() * sc[0, 0]).double().cpu()
        root += (v.float() * sc[0, 1]).double().cpu()
    for mean, want in ((total / 400, 0.5 * vals.double()), (root / 400, 0.5 * vals.double())):
        spacing = torch.maximum(want / 8, want.max() / 448 * 2.0 ** -9)
        assert ((mean - want).abs() <= 5 * 0.5 * spacing / 20 + 1e-7).all()


def test_8_bit_averages_follow_a_change():
    """After gradients shrink by 16, the 8-bit second moment of every element
    follows: 3000 steps at b2 = 0.999 leave 5% of the old one."""
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = AdamW([p], lr=0.0, state_bits=8, min_8bit_size=1)
    g = torch.Generator().manual_seed(0)
    size = torch.ones(n, device=DEV)
    for step in range(4000):
        if step == 1000:
            size[n // 2:] /= 16
            size[1::256] = 1.0                             # every block keeps a large element
        p.grad = size * (1 + 0.1 * torch.randn(n, generator=g)).to(DEV) if step % 50 == 0 else p.grad
        opt.step()
    s = opt.state[p]
    root = (s["root_avg_sq"].float().view(-1, 256) * s["scales"][:, 1:]).view(-1)
    small = size < 0.5
    want = float(((1 - 0.001) ** 3000 * 0.63 + (1 / 256) * 0.95) ** 0.5)
    got = float(root[small].square().mean().sqrt())
    assert 0.8 * want <= got <= 1.2 * want


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_follows_torchs(bits):
    """20 steps on a small network; float32 states: the parameters of torch's
    AdamW to 20 steps' roundings.  8-bit states: each step's direction is off
    by a code's spacing, at most 1/8 of a step's length."""
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(30, 80), torch.nn.Tanh(), torch.nn.Linear(80, 5)).to(DEV)
    twin = copy.deepcopy(net)
    groups = lambda n: [{"params": [n[0].weight, n[2].weight], "weight_decay": 0.1},  # noqa: E731
                        {"params": [n[0].bias, n[2].bias], "lr": 3e-3}]
    ours = AdamW(groups(net), lr=1e-3, state_bits=bits, min_8bit_size=1000)
    theirs = torch.optim.AdamW(groups(twin), lr=1e-3)
    x, y = torch.randn(64, 30, device=DEV), torch.randn(64, 5, device=DEV)
    for k in range(20):
        for n, o in ((net, ours), (twin, theirs)):
            o.zero_grad()
            if k == 7:                                     # a parameter without a gradient for once
                n[2].bias.requires_grad_(False)
            (n(x) - y).square().mean().backward()
            n[2].bias.requires_grad_(True)
            o.step()
    room = 1e-5 if bits == 32 else 20 * 3e-3 / 8
    for a, b in zip(net.parameters(), twin.parameters()):
        assert float((a - b).detach().abs().max()) <= room
    assert float(ours.state[net[2].bias]["step"]) == 19
    assert ("scales" in ours.state[net[0].weight]) == (bits == 8)
    assert "scales" not in ours.state[net[0].bias]


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(3000, device=DEV).bfloat16())
    opt = AdamW([p], state_bits=bits, min_8bit_size=1, seed=5)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    two = AdamW([q], state_bits=bits, min_8bit_size=1, seed=5)
    two.load_state_dict(copy.deepcopy(opt.state_dict()))
    for k, t in opt.state[p].items():
        assert two.state[q][k].dtype == t.dtype and torch.equal(two.state[q][k].float(), t.float())
    p.grad = torch.randn_like(p)
    q.grad = p.grad.clone()
    opt.step()
    two.step()
    assert torch.equal(p, q)


def test_layouts_and_python_path():
    base = torch.randn(8, 6, 5, 4, device=DEV)
    got = []
    for form, python in (("plain", False), ("last", False), ("last", True), ("plain", True)):
        fmt = torch.channels_last if form == "last" else torch.contiguous_format
        p = torch.nn.Parameter(base.clone().contiguous(memory_format=fmt))
        opt = AdamW([p], lr=1e-2, state_bits=8, min_8bit_size=1000)
        p.grad = (base * 0.3).contiguous()                 # another layout than the parameter's
        with _ext.python_path() if python else contextlib.nullcontext():
            opt.step()
        assert opt.state[p]["exp_avg"].stride() == p.stride()
        got.append(p.detach().clone())
    assert torch.equal(got[0], got[1]) and torch.equal(got[1], got[2]) and torch.equal(got[0], got[3])


def test_closure_and_captured_graph():
    p = torch.nn.Parameter(torch.randn(5000, device=DEV))
    lr = torch.tensor(1e-2, device=DEV)
    opt = AdamW([p], lr=lr)
    target = torch.randn(5000, device=DEV)

    def closure():
        opt.zero_grad()
        loss = (p - target).square().sum()
        loss.backward()
        return loss
    first = opt.step(closure)
    assert first.item() > 0
    q = torch.nn.Parameter(p.detach().clone())
    twin = torch.optim.AdamW([q], lr=1e-2)
    twin.load_state_dict({"state": {0: {k: v.clone() for k, v in opt.state[p].items()}},
                          "param_groups": twin.state_dict()["param_groups"]})
    grad = torch.zeros_like(p)
    p.grad = grad
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(graph, stream=s):
        opt.step()
    for k in range(5):
        grad.copy_(torch.randn(5000, device=DEV))
        lr.fill_(1e-2 / (k + 1))                           # a schedule inside the captured graph
        graph.replay()
        q.grad = grad.clone()
        twin.param_groups[0]["lr"] = 1e-2 / (k + 1)
        twin.step()
    assert float(opt.state[p]["step"]) == 6
    assert float((p - q).detach().abs().max()) <= 1e-5


def test_values_that_are_not_finite():
    """A NaN gradient spoils its own element (float32 states); in 8 bits also
    its block's states, and no other block's."""
    n = 1024
    g = torch.ones(n, device=DEV)
    g[300] = float("nan")
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(n, device=DEV))
        opt = AdamW([p], state_bits=bits, min_8bit_size=1)
        p.grad = g.clone()
        opt.step()
        assert torch.isnan(p).sum() == 1 and torch.isnan(p[300])
        p.grad = torch.ones(n, device=DEV)
        opt.step()
        bad = torch.isnan(p).nonzero()[:, 0].tolist()
        assert bad == ([300] if bits == 32 else list(range(256, 512)))
    p = torch.nn.Parameter(torch.ones(n, device=DEV))       # no gradient at all: only the decay
    opt = AdamW([p], lr=0.1, weight_decay=0.1, state_bits=8, min_8bit_size=1)
    p.grad = torch.zeros(n, device=DEV)
    opt.step()
    assert torch.allclose(p, torch.full_like(p, 0.99))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_overflowed_second_moment_stops_its_parameter(dtype):
    """g^2 beyond float32 with a finite first moment: the update is m / inf = 0,
    and only the decay is left (bound: three roundings of the parameter)."""
    p = torch.full((300,), 2.0, device=DEV, dtype=dtype)
    g = torch.zeros_like(p)
    g[7] = 1e25
    m, v, step = torch.zeros(300, device=DEV), torch.zeros(300, device=DEV), torch.zeros((), device=DEV)
    want = 2.0
    for _ in range(3):
        adamw_([p], [g], [m], [v], [step], lr=0.5, weight_decay=0.25)
        want *= 1.0 - 0.5 * 0.25
        assert torch.isinf(v[7]) and torch.isfinite(m[7])
        assert abs(p[7].item() - want) <= want * (3 * 3 * 2.0 ** -24 + 3 * ROUND[dtype])
        g[7] = 0.0


def test_refusals():
    def lists():
        z = lambda dt=F32, n=10: [torch.zeros(n, device=DEV, dtype=dt)]  # noqa: E731
        return dict(params=z(), grads=z(), exp_avgs=z(), exp_avg_sqs=z(), steps=[torch.zeros((), device=DEV)])
    z = torch.zeros
    for bad, kind in ((dict(grads=[z(9, device=DEV)]), ValueError),
                      (dict(grads=[z(10, device=DEV, dtype=BF16)]), TypeError),
                      (dict(exp_avgs=[z(10, device=DEV, dtype=F16)]), TypeError),
                      (dict(exp_avgs=[z(10, device=DEV, dtype=F8)]), TypeError),
                      (dict(exp_avgs=[z(10, device=DEV, dtype=F8)], exp_avg_sqs=[z(10, device=DEV, dtype=F8)]),
                       ValueError),
                      (dict(exp_avg_sqs=[z(10)]), RuntimeError),
                      (dict(steps=[z(1, device=DEV, dtype=torch.int64)]), TypeError),
                      (dict(params=[z(20, device=DEV)[::2]]), ValueError),
                      (dict(params=[z(10, device=DEV, dtype=torch.float64)],
                            grads=[z(10, device=DEV, dtype=torch.float64)]), TypeError),
                      (dict(steps=[]), ValueError),
                      (dict(betas=(0.9, 1.0)), _native.CpabNativeError)):
        for python in (False, True):
            with _ext.python_path() if python else contextlib.nullcontext():
                with pytest.raises(kind):
                    adamw_(**{**lists(), "lr": 1e-3, **bad})
    with pytest.raises(ValueError):
        adamw_(**lists(), lr=1e-3, workspace=torch.zeros(1, device=DEV))
    p = torch.nn.Parameter(torch.zeros(4, 4, device=DEV))
    p.grad = torch.zeros(4, 4, device=DEV).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW([p]).step()


def test_offsets_past_32_bits():
    n = (1 << 31) + 5000
    p = torch.zeros(n, device=DEV, dtype=BF16)
    g = torch.zeros(n, device=DEV, dtype=BF16)
    m, v = (torch.zeros(n, device=DEV, dtype=F8) for _ in range(2))
    sc = torch.zeros(-(-n // 256), 2, device=DEV)
    g[-300:] = 1
    adamw_([p], [g], [m], [v], [torch.zeros((), device=DEV)], scales=[sc], lr=1e-2, weight_decay=0.0)
    # the first step's length is lr whatever the gradient's size
    assert torch.allclose(p[-300:].float(), torch.full((300,), -1e-2, device=DEV), rtol=2 ** -8)
    assert not p[:-300].any() and math.isclose(float(sc[-1, 0]), 0.1 / 448, rel_tol=1e-6)
    assert (m[-300:].float() > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("python", [False, True])
def test_autograd_sees_the_step(bits, python):
    """As of torch's own in-place operations: a backward through a value that the
    step has replaced raises instead of using the new one."""
    p = torch.nn.Parameter(torch.randn(300, device=DEV))
    opt = AdamW([p], state_bits=bits, min_8bit_size=1)
    p.grad = torch.ones_like(p)
    with _ext.python_path() if python else contextlib.nullcontext():
        opt.step()
        old, normed = (p * p).sum(), rms_norm(torch.randn(3, 300, device=DEV), p).sum()
        written = [p, *opt.state[p].values()]
        before = [t._version for t in written]
        opt.step()
        assert all(t._version > n for t, n in zip(written, before))
        for loss in (old, normed):
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                loss.backward()
        with torch.inference_mode():                       # such tensors count no versions
            q, g, m, v = (torch.ones(10, device=DEV) for _ in range(4))
            step = torch.zeros((), device=DEV)
        adamw_([q], [g], [m], [v], [step], lr=1e-2)
        assert float(step) == 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_overflowed_second_moment_in_8_bits(dtype):
    """One gradient whose square overflows: its element only decays, the others of
    its block stay finite and the other blocks do not notice."""
    n, hyper = 700, dict(lr=0.5, weight_decay=0.25)
    g = torch.Generator().manual_seed(3)
    grads = torch.randn(6, n, generator=g).to(DEV, dtype)
    grads[1:, 300] = 0
    runs = []
    for size in (0.0, 1e25):
        p = torch.full((n,), 2.0, device=DEV, dtype=dtype)
        m, v = (torch.zeros(n, device=DEV, dtype=F8) for _ in range(2))
        sc, step, seen = torch.zeros(3, 2, device=DEV), torch.zeros((), device=DEV), []
        for k in range(6):
            grad = grads[k].clone()
            if k == 0:
                grad[300] = size
            adamw_([p], [grad], [m], [v], [step], scales=[sc], seed=4, **hyper)
            seen.append(p.clone())
        assert torch.isfinite(m.float()).all() and torch.isfinite(v.float()).all() and torch.isfinite(sc).all()
        runs.append(torch.stack(seen))
    plain, big = runs
    assert torch.isfinite(big).all()
    other = torch.ones(n, dtype=torch.bool, device=DEV)
    other[256:512] = False
    assert torch.equal(big[:, other], plain[:, other])
    mates = ~other
    mates[300] = False
    assert torch.equal(big[0, mates], plain[0, mates])
    want = 2.0
    for k in range(6):                                     # (as of the 32-bit states)
        want *= 1.0 - 0.5 * 0.25
        assert abs(big[k, 300].item() - want) <= want * (6 * 3 * 2.0 ** -24 + 6 * ROUND[dtype])


def test_an_8_bit_run_resumes_with_its_random_bits():
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(3000, device=DEV))
    opt = AdamW([p], state_bits=8, min_8bit_size=1, seed=5)
    p.grad = torch.randn_like(p)
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    two = AdamW([q], state_bits=8, min_8bit_size=1)
    two.load_state_dict(copy.deepcopy(opt.state_dict()))
    q.grad = p.grad.clone()
    opt.step()
    two.step()
    assert torch.equal(p, q)
    for k, t in opt.state[p].items():
        assert torch.equal(t.float(), two.state[q][k].float())


def test_groups_with_seeds_of_their_own():
    """A group's codes are those of an optimizer with its seed."""
    ps = [torch.nn.Parameter(torch.zeros(500, device=DEV)) for _ in range(3)]
    g = torch.randn(500, generator=torch.Generator().manual_seed(1)).to(DEV)
    for p in ps:
        p.grad = g.clone()
    kinds = dict(state_bits=8, min_8bit_size=1)
    both = AdamW([{"params": [ps[0]], "seed": 1}, {"params": [ps[1]], "seed": 2}], **kinds)
    one = AdamW([ps[2]], seed=2, **kinds)
    both.step()
    one.step()
    codes = lambda o, p: o.state[p]["exp_avg"].float()  # noqa: E731
    assert torch.equal(codes(both, ps[1]), codes(one, ps[2]))
    assert not torch.equal(codes(both, ps[0]), codes(both, ps[1]))


def test_copies_and_pickles_take_the_same_step():
    import io
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(700, device=DEV))
    opt = AdamW([p], state_bits=8, min_8bit_size=1, seed=5)
    for k in range(3):
        p.grad = torch.randn_like(p)
        opt.step()
    file = io.BytesIO()                                    # (torch pickles 8-bit tensors by its own save only)
    torch.save(opt, file)
    file.seek(0)
    two, three = copy.deepcopy(opt), torch.load(file, weights_only=False)
    grad = torch.randn_like(p)
    for o in (opt, two, three):
        (q,) = o.param_groups[0]["params"]
        q.grad = grad.clone()
        o.step()
    for o in (two, three):
        (q,) = o.param_groups[0]["params"]
        assert q is not p and torch.equal(p, q)
        for k, t in opt.state[p].items():
            assert torch.equal(t.float(), o.state[q][k].float())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_run_of_torchs_adamw_goes_on(dtype):
    """From its state dict.  float32: torch's parameters to the steps' roundings.
    bfloat16: torch rounds the moments too; a step is lr long at most, and each
    side rounds the parameter once a step."""
    torch.manual_seed(0)
    p = torch.nn.Parameter((0.1 * torch.randn(40, 30, device=DEV)).to(dtype))
    theirs = torch.optim.AdamW([p], lr=1e-3)
    for _ in range(3):
        p.grad = torch.randn_like(p)
        theirs.step()
    q = torch.nn.Parameter(p.detach().clone())
    ours = AdamW([q])
    ours.load_state_dict(theirs.state_dict())
    assert ours.state[q]["exp_avg"].dtype == F32
    for _ in range(5):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
        theirs.step()
        ours.step()
    assert float(ours.state[q]["step"]) == 8
    room = 1e-5 if dtype == F32 else 5 * (1e-3 + 2 * ROUND[dtype] * float(p.detach().abs().max()))
    assert float((p - q).detach().abs().max()) <= room


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_block_goes_from_tensor_to_tensor(dtype, bits):
    """130 tensors of odd sizes and 2300 chunks in one launch, so that a block's run
    holds chunks of several; a step count of each, two groups' hyperparameters."""
    sizes = [1 + (7919 * i) % 9000 for i in range(100)] + [1 + (104729 * i) % 300000 for i in range(30)]
    L = make(sizes, dtype, bits)
    old, cut = copies(L), 60
    other = dict(lr=5e-4, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.0)
    groups = []
    for part, h in ((slice(0, cut), HYPER), (slice(cut, None), other)):
        groups.append((*(L[k][part] for k in ("p", "g", "m", "v")), L["scales"][part] if bits == 8 else None,
                       L["step"][part], h["lr"], h["betas"], h["eps"], h["weight_decay"]))
    _step(groups, 9, torch.zeros(1, device=DEV, dtype=torch.int32))
    for part, h in ((range(cut), HYPER), (range(cut, len(sizes)), other)):
        check({k: [v[i] for i in part] for k, v in L.items()}, {k: [v[i] for i in part] for k, v in old.items()},
              dtype, 9, hyper=h, index=list(part))


def test_a_first_step_is_not_captured():
    """Its states' zeros would be part of the graph, and every replay a first step."""
    p = torch.nn.Parameter(torch.randn(300, device=DEV))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    assert float(opt.state[p]["step"]) == 4 and not torch.equal(p, before)


def test_loaded_states_step_first_in_a_capture():
    """What the capture allocates is not kept for the steps outside of it."""
    p = torch.nn.Parameter(torch.randn(300, device=DEV))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = p.grad.clone()
    two = AdamW([q])
    two.load_state_dict(opt.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two.step()
    assert not two._workspace
    two.step()
    graph.replay()
    graph.replay()
    two.step()
    for _ in range(4):
        opt.step()
    assert float(two.state[q]["step"]) == 5 and torch.equal(p, q)
