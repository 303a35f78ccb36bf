"""gated_scan and gated_scan_step against the recurrence sample by sample in
float64.

Tolerances (relative L2 over a tensor), from the arithmetic: a state's error
per step is a few float32 roundings (a, 1 - a, the multiply-add: 3 x 2^-24 of
the state's size) and fades with the state's own memory 1 / (1 - a), 23 samples
on average for the gates drawn here, so it grows like the root of half of that:
about 6e-7; 8 times that is allowed.  An output in 16 bits is off by at most
its unit roundoff on top.  Gradients carry two such chains: twice as much."""
import contextlib

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.recurrence import gated_scan, gated_scan_step

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
STATE = 5e-6
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # unit roundoffs: 11 and 8 significand bits


def tol(dtype, k=1):
    return k * STATE + ROUND[dtype]


def off(got, want):
    want = want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    d = torch.nan_to_num(got.double() - want)
    size = torch.nan_to_num(want).norm().clamp_min(1e-30)
    return (d.norm() / size).item() if want.numel() else 0.0


def reference(x, z, h0, lengths, dh=None, dlast=None):
    """float64, one sample at a time; NaN after a series' end must not matter."""
    B, T, D = x.shape
    x, z = x.double(), z.double()
    n = torch.full((B,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    live = (torch.arange(T, device=x.device)[None] < n[:, None])[..., None]
    one = torch.ones((), device=x.device, dtype=torch.float64)
    a = torch.where(live, torch.sigmoid(z), one)
    f = torch.where(live, torch.sigmoid(-z), 0 * one)
    x = torch.where(live, x, 0 * one)
    h = torch.zeros(B, D, device=x.device, dtype=torch.float64) if h0 is None else h0.double()
    start, hs = h, []
    for t in range(T):
        h = a[:, t] * h + f[:, t] * x[:, t]
        hs.append(h)
    H = torch.stack(hs, 1) if T else x
    out = torch.where(live, H, 0 * one)
    if dh is None and dlast is None:
        return out, h
    prev = torch.cat([start[:, None], H[:, :-1]], 1) if T else H
    c = torch.zeros_like(h) if dlast is None else dlast.double()
    g = torch.zeros_like(x) if dh is None else torch.where(live, dh.double(), 0 * one)
    delta = torch.zeros_like(x)
    for t in range(T - 1, -1, -1):
        delta[:, t] = g[:, t] + c
        c = a[:, t] * delta[:, t]
    dx = torch.where(live, f * delta, 0 * one)
    dz = torch.where(live, delta * (prev - x) * a * f, 0 * one)
    return out, h, dx, dz, c


def inputs(B, T, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, D, generator=g).to(DEV, dtype)
    z = (torch.randn(B, T, D, generator=g) * 1.5 + 2).to(DEV, dtype)
    h0 = torch.randn(B, D, generator=g).to(DEV)
    dh = torch.randn(B, T, D, generator=g).to(DEV, dtype)
    dl = torch.randn(B, D, generator=g).to(DEV)
    return x, z, h0, dh, dl


SHAPES = [(1, 1, 1), (3, 1, 40), (3, 17, 5), (2, 16, 2), (2, 64, 64), (2, 65, 66), (5, 301, 130),
          (1, 1000, 7), (4, 129, 257), (2, 2050, 96), (1, 5000, 16), (300, 3, 33)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_scan_and_gradient(shape, dtype, ragged):
    B, T, D = shape
    x, z, h0, dh, dl = inputs(B, T, D, dtype)
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(1)).int().to(DEV)
        lengths[0] = 0                                    # a series without a sample
    leaves = [t.requires_grad_(True) for t in (x, z, h0)]
    h, last = gated_scan(x, z, h0, lengths)
    grads = torch.autograd.grad((h, last), leaves, (dh, dl))
    ref = reference(x.detach(), z.detach(), h0.detach(), lengths, dh, dl)
    assert h.dtype == dtype and last.dtype == F32 and [g.dtype for g in grads] == [dtype, dtype, F32]
    assert off(h, ref[0]) <= tol(dtype) and off(last, ref[1]) <= tol(F32)
    for g, r, t in zip(grads, ref[2:], (dtype, dtype, F32)):
        assert off(g, r) <= tol(t, 2)
    with torch.no_grad():                                 # without a gradient: the same values
        h2, last2 = gated_scan(x, z, h0, lengths)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 70, 12), (3, 33, 9), (1, 700, 130)])
def test_packed_projection(shape, dtype):
    B, T, D = shape
    x, z, h0, dh, dl = inputs(B, T, D, dtype)
    xz = torch.cat([x, z], -1).requires_grad_(True)
    h, last = gated_scan(xz, h0=h0)
    (g,) = torch.autograd.grad((h, last), xz, (dh, dl))
    ref = reference(x, z, h0, None, dh, dl)
    assert off(h, ref[0]) <= tol(dtype) and off(last, ref[1]) <= tol(F32)
    assert off(g[..., :D], ref[2]) <= tol(dtype, 2) and off(g[..., D:], ref[3]) <= tol(dtype, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    B, T, D = 3, 150, 24
    x, z, h0, dh, dl = inputs(B, T, D, dtype)
    ref = reference(x, z, h0, None, dh, dl)
    wide = torch.zeros(B, T, 2 * D + 3, device=DEV, dtype=dtype)
    wide[..., 1:D + 1], wide[..., D + 2:2 * D + 2] = x, z
    forms = {
        "halves at odd offsets": (wide[..., 1:D + 1], wide[..., D + 2:2 * D + 2]),
        "time first": (x.transpose(0, 1).contiguous().transpose(0, 1), z),
        "channels first": (x.transpose(1, 2).contiguous().transpose(1, 2), z),
        "every second channel": (torch.stack([x, x], -1).flatten(2)[..., ::2], z),
    }
    for name, (a, b) in forms.items():
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        h, last = gated_scan(a, b, h0)
        ga, gb = torch.autograd.grad((h, last), (a, b), (dh, dl))
        assert off(h, ref[0]) <= tol(dtype), name
        assert off(ga, ref[2]) <= tol(dtype, 2) and off(gb, ref[3]) <= tol(dtype, 2), name
    # a broadcast gate: its gradient is summed over what it was broadcast to
    row = z[:1, :1].clone().requires_grad_(True)
    h, _ = gated_scan(x, row.expand(B, T, D), h0)
    (g,) = torch.autograd.grad(h, row, dh)
    r = reference(x, row.detach().expand(B, T, D), h0, None, dh, None)
    assert off(g, r[3].sum((0, 1), keepdim=True)) <= tol(dtype, 2) * 8  # a sum of 450 rounded terms
    # incoming gradients in any layout
    xg = x.detach().requires_grad_(True)
    h, last = gated_scan(xg, z, h0)
    (g1,) = torch.autograd.grad(h, xg, dh.transpose(0, 1).contiguous().transpose(0, 1), retain_graph=True)
    (g2,) = torch.autograd.grad(h.sum(), xg)
    assert off(g1, reference(x, z, h0, None, dh, None)[2]) <= tol(dtype, 2)
    assert off(g2, reference(x, z, h0, None, torch.ones_like(dh), None)[2]) <= tol(dtype, 2)


def test_one_gradient_at_a_time():
    x, z, h0, dh, dl = inputs(2, 100, 20, F32)
    for which in ("h", "last"):
        for leaf in range(3):
            t = [x.clone(), z.clone(), h0.clone()]
            t[leaf].requires_grad_(True)
            h, last = gated_scan(*t)
            (g,) = torch.autograd.grad(h if which == "h" else last, t[leaf], dh if which == "h" else dl)
            r = reference(x, z, h0, None, dh if which == "h" else None, dl if which == "last" else None)
            assert off(g, r[2 + leaf]) <= tol(F32, 2), (which, leaf)
    x.requires_grad_(True)
    h, _ = gated_scan(x, z)                               # h0 None: from zeros
    (g,) = torch.autograd.grad(h, x, dh)
    r = reference(x.detach(), z, None, None, dh, None)
    assert off(h, r[0]) <= tol(F32) and off(g, r[2]) <= tol(F32, 2)


def test_gradient_against_differences():
    """The directional derivative by central differences: with step 1e-2 the
    formula's third derivative leaves about 1e-4 of the slope, the float32
    values' noise (1e-6 of the sum, over 1e-2) about as much; 1e-2 is allowed."""
    x, z, h0, dh, dl = inputs(2, 90, 6, F32, seed=3)
    g = torch.Generator().manual_seed(5)
    leaves = [t.requires_grad_(True) for t in (x, z, h0)]
    h, last = gated_scan(*leaves)
    grads = torch.autograd.grad((h, last), leaves, (dh, dl))
    for leaf in range(3):
        u = torch.randn(leaves[leaf].shape, generator=g).to(DEV)
        sides = []
        for s in (1e-2, -1e-2):
            t = [v.detach().clone() for v in leaves]
            t[leaf] += s * u
            h, last = gated_scan(*t)
            sides.append((h.double() * dh).sum() + (last.double() * dl).sum())
        slope = float((sides[0] - sides[1]) / 2e-2)
        want = float((grads[leaf].double() * u).sum())
        assert abs(slope - want) <= 1e-2 * float(grads[leaf].norm()), leaf


def test_what_lies_after_a_series_does_not_matter():
    B, T, D = 4, 100, 10
    x, z, h0, dh, dl = inputs(B, T, D, F32)
    n = torch.tensor([0, 37, 100, 64], device=DEV, dtype=torch.int32)
    past = torch.arange(T, device=DEV)[None, :, None] >= n[:, None, None]
    ref = reference(x, z, h0, n, dh, dl)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(F32).min, torch.finfo(F32).max):
        t = [torch.where(past, torch.full_like(v, bad), v) for v in (x, z, dh)]
        leaves = [t[0].requires_grad_(True), t[1].requires_grad_(True), h0.clone().requires_grad_(True)]
        h, last = gated_scan(*leaves, lengths=n)
        grads = torch.autograd.grad((h, last), leaves, (t[2], dl))
        for got, want in zip((h, last, *grads), ref):
            assert off(got, want) <= tol(F32, 2)
        assert not h[past.expand_as(h)].any() and not grads[1][past.expand_as(h)].any()
    # lengths out of range are 0 and T; 64-bit ones are taken
    wild = torch.tensor([-5, 37, 2 ** 31 - 1, 64], device=DEV, dtype=torch.int32)
    assert torch.equal(gated_scan(x, z, h0, wild)[0], gated_scan(x, z, h0, n)[0])
    wild = torch.tensor([-2 ** 40, 37, 2 ** 40, 64], device=DEV)
    assert torch.equal(gated_scan(x, z, h0, wild)[0], gated_scan(x, z, h0, n)[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_gates_at_the_ends_of_their_type(dtype):
    """A gate at the type's lowest value or -inf takes the input, one at the
    highest or +inf keeps the state: exactly."""
    T, D = 40, 6
    x, _, h0, dh, _ = inputs(1, T, D, dtype)
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    for low, high in ((lo, hi), (-float("inf"), float("inf"))):
        z = torch.full((1, T, D), low, device=DEV, dtype=dtype)
        z[:, 10:] = high
        xg, zg = x.clone().requires_grad_(True), z.requires_grad_(True)
        h, last = gated_scan(xg, zg, h0)
        assert torch.equal(h[:, :10], x[:, :10])
        assert torch.equal(h[:, 10:], x[:, 9:10].expand(1, T - 10, D))
        assert torch.equal(last, x[:, 9].float())
        gx, gz = torch.autograd.grad(h, (xg, zg), dh)
        assert not gz.any() and not gx[:, 10:].any() and torch.equal(gx[:, :9], dh[:, :9])
    z = torch.zeros(1, T, D, device=DEV, dtype=dtype)
    z[0, 5, 2] = float("nan")                             # a NaN gate spoils its channel from there on
    h, last = gated_scan(x, z, h0)
    bad = torch.zeros(1, T, D, dtype=torch.bool, device=DEV)
    bad[0, 5:, 2] = True
    assert torch.equal(torch.isnan(h), bad) and torch.equal(torch.isnan(last), bad[:, -1])


def test_empty_sizes():
    for B, T, D in ((0, 5, 4), (3, 0, 4), (2, 3, 0)):
        x = torch.zeros(B, T, D, device=DEV, requires_grad=True)
        h0 = torch.randn(B, D, device=DEV, requires_grad=True)
        h, last = gated_scan(x, torch.zeros(B, T, D, device=DEV), h0)
        assert h.shape == (B, T, D) and last.shape == (B, D)
        if T == 0:
            assert torch.equal(last, h0)
            dl = torch.randn(B, D, device=DEV)
            assert torch.equal(torch.autograd.grad(last, h0, dl)[0], dl)
            assert not gated_scan(x.detach(), x.detach())[1].any()


def test_series_in_pieces_equal_the_whole():
    x, z, h0, _, _ = inputs(3, 333, 40, F32)
    want, end = gated_scan(x, z, h0)
    got, state = [], h0
    for a, b in ((0, 1), (1, 100), (100, 101), (101, 333)):
        h, state = gated_scan(x[:, a:b], z[:, a:b], state)
        got.append(h)
    assert off(torch.cat(got, 1), want) <= tol(F32) and off(state, end) <= tol(F32)
    state = h0.clone()
    for t in range(20):
        h = gated_scan_step(x[:, t], z[:, t], state)
        assert off(h, want[:, t]) <= tol(F32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,D,rows", [(1, 1, 1), (5, 7, 9), (64, 512, 96), (33, 130, 33)])
@pytest.mark.parametrize("packed", [False, True])
def test_step(B, D, rows, dtype, packed):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(B, D, generator=g).to(DEV, dtype)
    z = (torch.randn(B, D, generator=g) * 2 + 1).to(DEV, dtype)
    state = torch.randn(rows, D, generator=g).to(DEV)
    slots = torch.randperm(rows, generator=g)[:B].int().to(DEV)
    slots[B // 2:B // 2 + 1] = -1
    if B > 4:
        slots[3] = rows                                   # past the table: no stream either
    before = state.clone()
    args = (torch.cat([x, z], 1), None) if packed else (x, z)
    h = gated_scan_step(*args, state, slots)
    want, out = before.double(), torch.zeros(B, D, dtype=torch.float64, device=DEV)
    for b, s in enumerate(slots.tolist()):
        if 0 <= s < rows:
            want[s] = torch.sigmoid(z[b].double()) * want[s] + torch.sigmoid(-z[b].double()) * x[b].double()
            out[b] = want[s]
    assert off(state, want) <= tol(F32) and off(h, out) <= tol(dtype)
    idle = torch.ones(rows, dtype=torch.bool, device=DEV)
    idle[[s for s in slots.tolist() if 0 <= s < rows]] = False
    assert torch.equal(state[idle], before[idle])


def test_python_path_is_the_same():
    x, z, h0, dh, dl = inputs(3, 150, 22, BF16)
    n = torch.tensor([150, 0, 77], device=DEV)
    got = []
    for python in (False, True):
        leaves = [t.clone().requires_grad_(True) for t in (x, z, h0)]
        state = h0.clone()
        xz = torch.cat([x, z], -1).requires_grad_(True)
        import contextlib
        with _ext.python_path() if python else contextlib.nullcontext():
            h, last = gated_scan(*leaves, lengths=n)
            grads = torch.autograd.grad((h, last), leaves, (dh, dl))
            hp, _ = gated_scan(xz)
            gp = torch.autograd.grad(hp, xz, dh)
            s = gated_scan_step(x[:, 0], z[:, 0], state, torch.tensor([2, -1, 0], device=DEV))
        got.append((h, last, *grads, hp, *gp, s, state))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_another_stream_and_a_captured_graph():
    x, z, h0, dh, dl = inputs(2, 400, 64, F32)
    want = gated_scan(x, z, h0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = gated_scan(x, z, h0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    xs = x.clone().requires_grad_(True)

    def step():
        h, last = gated_scan(xs, z, h0)
        return (h, last, *torch.autograd.grad((h, last), xs, (dh, dl)))
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        xs.copy_(x * 2)
    graph.replay()
    for a, b in zip(out, reference(x * 2, z, h0, None, dh, dl)):
        assert off(a, b) <= tol(F32, 2)


def test_long_series_in_pieces():
    """Few channels, many samples: blocks that take pieces of one series, on
    another stream, in a captured graph, and with a NaN that reaches the end."""
    x, z, h0, dh, dl = inputs(1, 6000, 24, BF16, seed=9)
    n = torch.tensor([5900], device=DEV, dtype=torch.int32)
    xs = x.clone().requires_grad_(True)

    def step():
        h, last = gated_scan(xs, z, h0, n)
        return (h, last, *torch.autograd.grad((h, last), xs, (dh, dl)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first = step()
    torch.cuda.current_stream().wait_stream(s)
    ref = reference(x, z, h0, n, dh, dl)
    for got, want, t in zip(first, ref, (BF16, F32, BF16)):
        assert off(got, want) <= tol(t, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        xs.copy_(x * 2)
    for _ in range(3):
        graph.replay()
    for got, want, t in zip(out, reference(x * 2, z, h0, n, dh, dl), (BF16, F32, BF16)):
        assert off(got, want) <= tol(t, 2)
    x[0, 100, 3] = float("nan")
    h, last = gated_scan(x, z, h0, n)
    bad = torch.zeros(6000, 24, dtype=torch.bool, device=DEV)
    bad[100:5900, 3] = True
    assert torch.equal(torch.isnan(h[0]), bad) and torch.equal(torch.isnan(last[0]), bad[5899])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("channels", [512, 509])
@pytest.mark.parametrize("length", [640, 1111])
def test_one_or_two_tiles_on_an_sm(dtype, channels, length):
    """Tiles enough for a GPU's SMs but not for several on each: wide blocks,
    whole and ragged, rows on and off 16 bytes."""
    B = 10 if dtype == F32 else 12                        # 150 to 320 tiles
    D = channels if dtype != F32 else channels // 2
    x, z, h0, dh, dl = inputs(B, length, D, dtype, seed=11)
    n = torch.randint(0, length + 1, (B,), generator=torch.Generator().manual_seed(2)).int().to(DEV)
    n[:4] = torch.tensor([0, 1, length, length - 1], dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (x, z, h0)]
    h, last = gated_scan(x, z, h0, n)
    grads = torch.autograd.grad((h, last), leaves, (dh, dl))
    ref = reference(x.detach(), z.detach(), h0.detach(), n, dh, dl)
    assert off(h, ref[0]) <= tol(dtype) and off(last, ref[1]) <= tol(F32)
    for g, r, t in zip(grads, ref[2:], (dtype, dtype, F32)):
        assert off(g, r) <= tol(t, 2)


def test_the_python_node_refuses_a_second_gradient_too():
    x, z, h0, _, _ = inputs(2, 9, 8, F32)
    x.requires_grad_(True)
    with _ext.python_path():
        h, _ = gated_scan(x, z, h0)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad((h * x).sum(), x, create_graph=True)
        torch.autograd.grad((h * x).sum(), x)


def test_refusals():
    x = torch.zeros(2, 5, 4, device=DEV)
    with pytest.raises(ValueError):
        gated_scan(x[0], x[0])
    with pytest.raises(ValueError):
        gated_scan(x, x[..., :3])
    with pytest.raises(ValueError):
        gated_scan(x[..., :3])
    with pytest.raises(TypeError):
        gated_scan(x, x.bfloat16())
    with pytest.raises(TypeError):
        gated_scan(x.double(), x.double())
    with pytest.raises(TypeError):
        gated_scan(x, x, h0=torch.zeros(2, 4, device=DEV, dtype=BF16))
    with pytest.raises(ValueError):
        gated_scan(x, x, h0=torch.zeros(2, 3, device=DEV))
    with pytest.raises(ValueError):
        gated_scan(x, x, lengths=torch.zeros(3, device=DEV, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        gated_scan(x, x, lengths=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        gated_scan_step(x[:, 0], x[:, 0], torch.zeros(3, 4, device=DEV))
    with pytest.raises(ValueError):
        gated_scan_step(x[:, 0], x[:, 0], torch.zeros(4, 2, device=DEV).t(), torch.zeros(2, device=DEV).int())
    h, _ = gated_scan(x.requires_grad_(True), x)
    with pytest.raises(RuntimeError, match="once|differentiable"):
        g = torch.autograd.grad(h.sum(), x, create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(_native.CpabNativeError, match="2\\^30"):
        gated_scan(torch.zeros(1, 1, 1, device=DEV).expand(1 << 20, 1, 1 << 11),
                   torch.zeros(1, 1, 1, device=DEV).expand(1 << 20, 1, 1 << 11))


def test_offsets_past_32_bits():
    """2.2e9 elements; short memory, so the end can be checked from nearby."""
    T, D = (1 << 20) + 77, 2112
    x = torch.empty(1, T, D, device=DEV, dtype=BF16).normal_()
    z = torch.zeros(1, T, D, device=DEV, dtype=BF16)
    x.requires_grad_(True)
    z.requires_grad_(True)
    h, last = gated_scan(x, z)
    k = 300                                               # 2^-200: nothing is left of what was before
    tail = [t[:, -k:].detach().clone() for t in (x, z)]
    dh = torch.zeros_like(h)
    dh[:, -100:] = 1
    gx, gz = torch.autograd.grad(h, (x, z), dh)
    r = reference(*tail, None, None, dh[:, -k:], None)
    assert off(h[:, -100:], r[0][:, -100:]) <= tol(BF16) and off(last, r[1]) <= tol(F32)
    assert off(gx[:, -150:], r[2][:, -150:]) <= tol(BF16, 2)
    assert off(gz[:, -150:], r[3][:, -150:]) <= tol(BF16, 2)


@pytest.mark.parametrize("python", [False, True])
def test_autograd_sees_the_step_of_a_state(python):
    """A backward through the old state raises instead of using the new one."""
    x, z, _, _, _ = inputs(4, 1, 10, F32)
    w = torch.ones(4, 10, device=DEV, requires_grad=True)
    state = torch.randn(2, 4, 10, device=DEV)
    with _ext.python_path() if python else contextlib.nullcontext():
        loss = (w * state[1]).sum()
        gated_scan_step(x[:, 0], z[:, 0], state[1])
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()
        with torch.inference_mode():                       # such tensors count no versions
            state = torch.zeros(4, 10, device=DEV)
        h = gated_scan_step(x[:, 0], z[:, 0], state)
        assert torch.equal(h, state)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(python, grad):
    """Instead of coming out as none."""
    from torch.autograd import forward_ad
    x, z, h0, _, _ = inputs(2, 9, 8, F32)
    with (_ext.python_path() if python else contextlib.nullcontext()), torch.set_grad_enabled(grad), \
            forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), z, h0), (x, dual(z), h0), (x, z, dual(h0))):
            with pytest.raises(RuntimeError, match="jvp|forward"):
                gated_scan(*args)
        for args in ((dual(x[:, 0]), z[:, 0], h0), (x[:, 0], dual(z[:, 0]), h0), (x[:, 0], z[:, 0], dual(h0))):
            with pytest.raises(RuntimeError, match="no gradient"):
                gated_scan_step(*args)
        gated_scan(x, z, h0)


def test_float32_gates_keep_their_relative_precision():
    """a and 1 - a of gates up to 40 against float64.  Bound: the exponential
    instruction's 2^-22, 2e-9 x 58 left of its argument, 2^-23 of the reciprocal and
    four roundings (the correction, 1 + e, e a and, of dz, one product): 7e-7; dz,
    a product of both, twice that."""
    z = torch.linspace(-40, 40, 1 << 14, device=DEV)
    one, none = torch.ones_like(z), torch.zeros_like(z)
    a, f = torch.sigmoid(z.double()), torch.sigmoid(-z.double())

    def close(got, want, k=1):
        return float((got.detach().double() / want - 1).abs().max()) <= k * 7e-7
    # one sample (a thread per channel), and the first of 40 whose others change nothing (tiles)
    for T in (1, 40):
        def series(first, rest):
            return torch.cat([first[None, None], torch.full((1, T - 1, z.numel()), rest, device=DEV)], 1)
        for x, h0, want in ((one, none, f), (none, one, a)):
            xs, zs = series(x, 0.0).requires_grad_(True), series(z, float("inf")).requires_grad_(True)
            hs = h0[None].clone().requires_grad_(True)
            h, last = gated_scan(xs, zs, hs)
            assert close(h[0, 0], want) and close(last[0], want), T
            gx, gz, gh = torch.autograd.grad(last, (xs, zs, hs), one[None])
            assert close(gx[0, 0], f) and close(gh[0], a), T
            assert close(gz[0, 0], a * f * (1.0 if h0 is one else -1.0), 2), T
    state = one[None].clone()
    assert close(gated_scan_step(none[None], z[None], state)[0], a)
    state.zero_()
    assert close(gated_scan_step(one[None], z[None], state)[0], f)


@pytest.mark.parametrize("shift", [7.0, 12.0])
@pytest.mark.parametrize("length", [8192, 63])
def test_long_memories(shift, length):
    """Gates of memories of a thousand samples: in float32 the states are as near to
    float64 as the recursion in elementary float32 operations is; twice that is
    allowed.  Of memories longer than the series that holds sample by sample only:
    composed steps multiply factors (1 - j u)(1 - k u), whose j k u^2 is always
    rounded away, so the head's bound for a memory of `length` samples is taken."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(2, length, 64, generator=g).to(DEV)
    z = (torch.randn(2, length, 64, generator=g) * 1.5 + shift).to(DEV)
    want, _ = reference(x, z, None, None)
    a, f, h, plain = torch.sigmoid(z), torch.sigmoid(-z), torch.zeros(2, 64, device=DEV), []
    for t in range(length):
        h = a[:, t] * h + f[:, t] * x[:, t]
        plain.append(h)
    room = 2 * off(torch.stack(plain, 1), want) if shift == 7 else 8 * 3 * 2.0 ** -24 * (length / 2) ** 0.5
    assert off(gated_scan(x, z)[0], want) <= room
    state = torch.zeros(2, 64, device=DEV)
    for t in range(length):
        h = gated_scan_step(x[:, t], z[:, t], state)
    assert off(h, want[:, -1]) <= 2 * off(plain[-1], want[:, -1])
