"""rms_norm and rms_norm_quantized against their formulas in float64.

Tolerances (relative L2 over a tensor): a value is a few float32 roundings
from exact, and so is the gradient (its subtraction leaves a part as large as
the rows' gradients); 1e-6 is 16 of them.  The weight's gradient sums rows of
random sign: as many roundings as the sum itself grows, 2e-6.  Outputs in 16
bits are off by at most their unit roundoff on top."""
import contextlib

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.norm import rms_norm, rms_norm_quantized

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROUND = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # unit roundoffs: 11 and 8 significand bits
EPS = 1e-6


def off(got, want):
    assert got.shape == want.shape
    d = got.double() - want.double()
    return (d.norm() / want.double().norm().clamp_min(1e-30)).item() if want.numel() else 0.0


def reference(x, w, res, eps=EPS, dy=None, ds=None):
    s = x.double() if res is None else (x.float() + res.float()).to(res.dtype).double()
    v, wd = s.clone().requires_grad_(True), w.detach().double().requires_grad_(True)
    y = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * wd
    if dy is None:
        return y.detach(), s
    gv, gw = torch.autograd.grad(y, (v, wd), dy.double())
    return y.detach(), s, gv if ds is None else gv + ds.double(), gw


def inputs(n, D, dtype, stream, wtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, D, generator=g).to(DEV, dtype)
    res = (2 * torch.randn(n, D, generator=g)).to(DEV, stream)
    w = (1 + 0.1 * torch.randn(D, generator=g)).to(DEV, wtype)
    dy = torch.randn(n, D, generator=g).to(DEV, dtype)
    ds = torch.randn(n, D, generator=g).to(DEV, stream)
    return x, res, w, dy, ds


SHAPES = [(1, 1), (3, 2), (700, 5), (5, 31), (33, 64), (515, 1000), (9, 1024), (130, 1537), (4, 4096),
          (700, 520), (2, 8192), (3, 16383), (2, 16384), (1500, 96)]
TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_with_residual(shape, types):
    dtype, stream, wtype = types
    x, res, w, dy, ds = inputs(*shape, *types)
    leaves = [t.requires_grad_(True) for t in (x, w, res)]
    y, s = rms_norm(x, w, residual=res, eps=EPS)
    gx, gw, gr = torch.autograd.grad((y, s), leaves, (dy, ds))
    ry, rs, rg, rw = reference(x.detach(), w, res.detach(), EPS, dy, ds)
    assert (y.dtype, s.dtype, gx.dtype, gr.dtype, gw.dtype) == (dtype, stream, dtype, stream, wtype)
    assert torch.equal(s.double(), rs)
    assert off(y, ry) <= 1e-6 + ROUND[dtype]
    assert off(gx, rg) <= 1e-6 + ROUND[dtype] and off(gr, rg) <= 1e-6 + ROUND[stream]
    assert off(gw, rw) <= 2e-6 + ROUND[wtype]
    with torch.no_grad():
        y2, s2 = rms_norm(x, w, residual=res, eps=EPS)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    again = torch.autograd.grad(rms_norm(x, w, residual=res, eps=EPS), leaves, (dy, ds))
    assert all(torch.equal(a, b) for a, b in zip(again, (gx, gw, gr)))    # the same every run


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_alone(shape, dtype):
    x, _, w, dy, _ = inputs(*shape, dtype, dtype, F32)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = rms_norm(x, w, eps=EPS)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    ry, _, rg, rw = reference(x.detach(), w, None, EPS, dy)
    # a row of one column: the gradient is what cancels, eps / x^2 of its terms
    grain = 1e-6 if shape[1] > 1 else 1.0
    assert off(y, ry) <= 1e-6 + ROUND[dtype] and off(gw, rw) <= 2e-6
    assert off(gx, rg) <= grain + ROUND[dtype]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_quantized(shape, types, residual):
    """A code stands for a value at most half a code's spacing away: 1/16 of
    the value, or scale / 1024 where codes are spaced evenly; 1e-5 of the row's
    largest value for the float32 values before."""
    dtype, stream, wtype = types
    x, res, w, _, _ = inputs(*shape, *types)
    res = res if residual else None
    out = rms_norm_quantized(x, w, residual=res, eps=EPS)
    q, scale = out[:2]
    ry, rs = reference(x, w, res, EPS)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == F32 and scale.shape == shape[:1]
    if residual:
        assert torch.equal(out[2].double(), rs) and out[2].dtype == stream
    top = ry.abs().amax(1)
    assert ((scale.double() - top / 448).abs() <= 1e-6 * top / 448).all()
    v = q.double() * scale.double()[:, None]
    assert torch.isfinite(v).all()
    room = torch.maximum(ry.abs() / 16, scale.double()[:, None] / 1024) + 1e-5 * top[:, None]
    assert ((v - ry).abs() <= room).all()
    assert (q.float().abs().amax(1) == 448).all()


def test_rows_of_zeros_and_extremes():
    D = 300
    x = torch.zeros(6, D, device=DEV)
    x[1], x[2, 7], x[3, 5], x[4] = 1e-30, float("nan"), 1e-18, 3e38
    w = torch.ones(D, device=DEV)
    y = rms_norm(x, w)
    q, scale = rms_norm_quantized(x, w)
    assert not y[0].any() and not q[0].float().any() and scale[0] == 2.0 ** -126
    assert torch.isnan(y[2]).all() and torch.isnan(scale[2])
    assert torch.isfinite(y[[0, 1, 3]]).all()
    assert off(y[1:2], x[1:2].double() * 1e3) <= 1e-5     # far below eps: x / sqrt(eps)
    assert not y[4].any()                                  # its mean square is past float32: r is 0
    one = torch.full((1, D), 2.0, device=DEV, dtype=BF16)
    assert torch.equal(rms_norm(one, w, eps=0.0), torch.ones_like(one))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shapes_strides_and_alignment(dtype):
    x, res, w, dy, ds = inputs(60, 48, dtype, dtype, F32)
    want = reference(x, w, res, EPS, dy, ds)
    wide = torch.zeros(60, 101, device=DEV, dtype=dtype)
    wide[:, 1:49], wide[:, 51:99] = x, res
    shaped = (3, 4, 5, 48)
    forms = {
        "rows at odd offsets": (wide[:, 1:49], wide[:, 51:99]),
        "columns first": (x.t().contiguous().t(), res),
        "four axes": (x.view(shaped), res.view(shaped)),
        "axes in another order": (x.view(shaped).permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3),
                                  res.view(shaped)),
        "every second row": (torch.stack([x, x], 1).flatten(0, 1)[::2], res),
    }
    for name, (a, b) in forms.items():
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        y, s = rms_norm(a, w, residual=b, eps=EPS)
        ga, gb = torch.autograd.grad((y, s), (a, b), (dy.view(a.shape), ds.view(a.shape)))
        assert y.shape == a.shape
        assert off(y.reshape(60, 48), want[0]) <= 1e-6 + ROUND[dtype], name
        assert off(ga.reshape(60, 48), want[2]) <= 1e-6 + ROUND[dtype], name
        assert off(gb.reshape(60, 48), want[2]) <= 1e-6 + ROUND[dtype], name
    off_w = torch.zeros(49, device=DEV)
    off_w[1:] = w
    assert off(rms_norm(x, off_w[1:], residual=res, eps=EPS)[0], want[0]) <= 1e-6 + ROUND[dtype]
    # one row for all: its gradient is the rows' sum
    one = res[:1].detach().clone().requires_grad_(True)
    y, s = rms_norm(x, w, residual=one.expand(60, 48), eps=EPS)
    (g,) = torch.autograd.grad((y, s), one, (dy, ds))
    r = reference(x, w, one.detach().expand(60, 48), EPS, dy, ds)
    assert off(g, r[2].sum(0, keepdim=True)) <= 8 * (1e-6 + ROUND[dtype])


def test_one_output_at_a_time():
    for types in ((F32, F32, F32), (BF16, F32, F32)):
        x, res, w, dy, ds = inputs(20, 40, *types)
        leaves = [t.requires_grad_(True) for t in (x, res, w)]
        y, s = rms_norm(x, w, residual=res, eps=EPS)
        gx, gr, gw = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        _, _, rg, rw = reference(x.detach(), w, res.detach(), EPS, dy, None)
        assert off(gx, rg) <= 1e-6 + ROUND[types[0]] and off(gr, rg) <= 1e-6 and off(gw, rw) <= 2e-6
        gx, gr, gw = torch.autograd.grad(s, leaves, ds, allow_unused=True)
        assert torch.equal(gx, ds.to(types[0])) and torch.equal(gr, ds) and (gw is None or not gw.any())
        frozen = w.detach()
        y, s = rms_norm(x, frozen, residual=res, eps=EPS)
        gx2, = torch.autograd.grad(y, x, dy)
        assert off(gx2, rg) <= 1e-6 + ROUND[types[0]]


def test_gradient_against_differences():
    """Central differences with step 1e-2: about 1e-4 of the slope is left of
    the third derivative, as much of the float32 noise; 1e-2 is allowed."""
    x, res, w, dy, ds = inputs(12, 30, F32, F32, F32, seed=4)
    g = torch.Generator().manual_seed(5)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    grads = torch.autograd.grad(rms_norm(x, w, residual=res), leaves, (dy, ds))
    for k in range(3):
        u = torch.randn(leaves[k].shape, generator=g).to(DEV)
        sides = []
        for step in (1e-2, -1e-2):
            t = [v.detach().clone() for v in leaves]
            t[k] += step * u
            y, s = rms_norm(t[0], t[2], residual=t[1])
            sides.append((y.double() * dy).sum() + (s.double() * ds).sum())
        slope = float((sides[0] - sides[1]) / 2e-2)
        assert abs(slope - float((grads[k].double() * u).sum())) <= 1e-2 * float(grads[k].norm()), k


def test_empty_and_python_path():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    y = rms_norm(x, w)
    assert y.shape == (0, 8) and not torch.autograd.grad(y.sum(), w)[0].any()
    with torch.no_grad():
        q, scale = rms_norm_quantized(x, w)
    assert q.shape == (0, 8) and scale.shape == (0,)
    for types in TYPES:
        x, res, w, dy, ds = inputs(37, 72, *types)
        got = []
        for python in (False, True):
            with _ext.python_path() if python else contextlib.nullcontext():
                leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, res)]
                y, s = rms_norm(*leaves[:2], residual=leaves[2])
                grads = torch.autograd.grad((y, s), leaves, (dy, ds))
                with torch.no_grad():
                    q = rms_norm_quantized(*leaves[:2], residual=leaves[2])
                got.append((y, s, *grads, *(t.float() for t in q)))
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_refusals():
    x, w = torch.zeros(3, 8, device=DEV), torch.ones(8, device=DEV)
    for args, kind in (((x, w[:7]), ValueError), ((x, w.bfloat16()), TypeError), ((x.double(), w), TypeError),
                       ((x, w, x[:2]), ValueError), ((x, w, x.half()), TypeError),
                       ((x.half(), w, x.bfloat16()), TypeError), ((x[:, :0], w[:0]), ValueError),
                       ((x, w.cpu()), RuntimeError)):
        with pytest.raises(kind):
            rms_norm(*args)
        with pytest.raises(kind):
            rms_norm_quantized(*args)
    with pytest.raises(_native.CpabNativeError, match="16384"):
        rms_norm(torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV))
    with pytest.raises(_native.CpabNativeError, match="eps"):
        rms_norm(x, w, eps=-1.0)
    y = rms_norm(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="once|differentiable"):
        g = torch.autograd.grad(y.sum(), x, create_graph=True)[0]
        torch.autograd.grad(g.sum(), x)


def test_the_python_node_refuses_a_second_gradient_too():
    x, w = torch.ones(3, 8, device=DEV, requires_grad=True), torch.ones(8, device=DEV)
    with _ext.python_path():
        y = rms_norm(x, w)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad((y * x).sum(), x, create_graph=True)
        torch.autograd.grad((y * x).sum(), x)


def test_offsets_past_32_bits():
    n, D = (1 << 17) + 5, 16384
    x = torch.empty(n, D, device=DEV, dtype=BF16).normal_()
    w = torch.ones(D, device=DEV)
    x.requires_grad_(True)
    y = rms_norm(x, w)
    dy = torch.zeros_like(x)
    dy[-3:] = 1
    (g,) = torch.autograd.grad(y, x, dy)
    ry, _, rg, _ = reference(x[-3:].detach(), w, None, EPS, dy[-3:])
    assert off(y[-3:], ry) <= 1e-6 + ROUND[BF16] and off(g[-3:], rg) <= 1e-6 + ROUND[BF16]
    assert not g[:-3].any()


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(python, grad):
    """Instead of coming out as none."""
    from torch.autograd import forward_ad
    x, res, w, _, _ = inputs(5, 8, F32, F32, F32)
    with (_ext.python_path() if python else contextlib.nullcontext()), torch.set_grad_enabled(grad), \
            forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), w, res), (x, dual(w), res), (x, w, dual(res)), (dual(x), w)):
            with pytest.raises(RuntimeError, match="jvp|forward"):
                rms_norm(*args)
            with pytest.raises(RuntimeError, match="no gradient"):
                rms_norm_quantized(*args)
        rms_norm(x, w, res)
        rms_norm_quantized(x, w, res)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_overlap(dtype):
    """Windows of one signal, a row a step of 1 or 8 further on: nothing lies
    between or after them."""
    for step, D in ((1, 33), (8, 40), (8, 48), (1, 41)):
        signal = torch.randn(400, generator=torch.Generator().manual_seed(2)).to(DEV, dtype)
        x = signal.unfold(0, D, step).detach().requires_grad_(True)
        _, res, w, dy, ds = inputs(x.shape[0], D, dtype, dtype, F32)
        y, s = rms_norm(x, w, residual=res, eps=EPS)
        (g,) = torch.autograd.grad((y, s), x, (dy, ds))
        want = reference(x.detach(), w, res, EPS, dy, ds)
        assert off(y, want[0]) <= 1e-6 + ROUND[dtype] and off(g, want[2]) <= 1e-6 + ROUND[dtype]
        y = rms_norm(x, w, eps=EPS)
        (g,) = torch.autograd.grad(y, x, dy)
        want = reference(x.detach(), w, None, EPS, dy)
        assert off(y, want[0]) <= 1e-6 + ROUND[dtype] and off(g, want[2]) <= 1e-6 + ROUND[dtype]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(7013, 999), (5003, 1537), (5003, 1024), (60013, 33), (1201, 9001)])
def test_many_rows_for_each_thread(shape, types):
    """More rows than the gradient's blocks hold at once, on vectors and inside
    them: the weight's gradient summed over rows (of random sign, so its error
    grows as it does)."""
    x, res, w, dy, ds = inputs(*shape, *types)
    leaves = [t.requires_grad_(True) for t in (x, w, res)]
    y, s = rms_norm(x, w, residual=res, eps=EPS)
    gx, gw, gr = torch.autograd.grad((y, s), leaves, (dy, ds))
    ry, rs, rg, rw = reference(x.detach(), w, res.detach(), EPS, dy, ds)
    assert torch.equal(s.double(), rs) and off(y, ry) <= 1e-6 + ROUND[types[0]]
    assert off(gx, rg) <= 1e-6 + ROUND[types[0]] and off(gr, rg) <= 1e-6 + ROUND[types[1]]
    assert off(gw, rw) <= 2e-6 + ROUND[types[2]]
    last = off(gx[-50:], rg[-50:])                         # (a row by itself hardly shows in the whole)
    assert last <= 1e-6 + ROUND[types[0]]
    with torch.no_grad():
        q, scale, _ = rms_norm_quantized(x, w, residual=res, eps=EPS)
    top = ry.abs().amax(1)
    assert ((scale.double() - top / 448).abs() <= 1e-6 * top / 448).all()
    v = q.double() * scale.double()[:, None]
    room = torch.maximum(ry.abs() / 16, scale.double()[:, None] / 1024) + 1e-5 * top[:, None]
    assert ((v - ry).abs() <= room).all()


def test_an_8_bit_scale_is_rounded_once():
    """Rows of ones and minus ones: r is 1, y the weights, the scale the float32
    nearest to their largest magnitude / 448."""
    g = torch.Generator().manual_seed(6)
    x = torch.where(torch.rand(64, 256, generator=g) < 0.5, -1.0, 1.0).to(DEV)
    for _ in range(40):
        w = torch.randn(256, generator=g)
        assert torch.equal(rms_norm(x, w.to(DEV), eps=0.0), x * w.to(DEV))
        _, scale = rms_norm_quantized(x, w.to(DEV), eps=0.0)
        want = (w.abs().max().double() / 448).float()
        assert torch.equal(scale.cpu(), want.expand(64))
