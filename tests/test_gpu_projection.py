"""quantize_blocks, matmul_quantized and linear_quantized against their
definitions in float64.

Codes and scales are exact: x over a power of two is exact and rounded once.

Products: a code product is exact; what is summed is cut to float32 (by less
than 2^-23 of what has been summed so far) at most once for each of the 32
codes that an instruction takes, so an element is off by at most
(K / 32 + 4) 2^-22 sum |x w| (a factor 2 covers the alignment of the 32
products among themselves), then by three float32 roundings of scales and bias
and half a step of the result's type."""
import contextlib

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.norm import rms_norm_quantized
from cpab.pytorch.projection import linear_quantized, matmul_quantized, quantize_blocks

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def two_to(e):
    return ((e + 1023) << 52).view(torch.float64)


def encoded(x):
    """Codes' values over the scale, and the scales' exponents, of a matrix."""
    R, K = x.shape
    nb = -(-K // 128)
    p = torch.zeros(R, nb * 128, device=x.device, dtype=torch.float64)
    p[:, :K] = x.double()
    p = p.view(R, nb, 128)
    m, k = torch.frexp(p.abs().amax(2))                  # amax = m 2^k; 448 = 0.875 2^9
    e = (k.long() - 9 + (m > 0.875)).clamp_min(-126)
    e = torch.where(p.abs().amax(2) == 0, -126, e)
    q = (p * two_to(-e)[..., None]).float().to(CODES)
    return q.view(R, nb * 128)[:, :K], e


def valued(q, e):
    return q.double() * torch.repeat_interleave(two_to(e), 128, 1)[:, :q.shape[1]]


def same_codes(q, scale, x):
    want, e = encoded(x)
    assert torch.equal(scale.view(torch.uint8).long(), e + 127)
    assert torch.equal(q.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


def features(R, K, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, K, generator=g) * torch.exp(spread * torch.randn(K, generator=g))).to(DEV, dtype)


@pytest.fixture(params=["ext", "python"])
def path(request):
    with _ext.python_path() if request.param == "python" else contextlib.nullcontext():
        yield request.param


SHAPES = [(1, 1), (1, 128), (3, 129), (16, 2048), (130, 7), (128, 16), (300, 1000), (515, 257), (1029, 384)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_codes(shape, dtype, path):
    x = features(*shape, dtype)
    q, s, qt, st = quantize_blocks(x, transposed=True)
    assert q.dtype == CODES and s.dtype == SCALES and q.shape == x.shape and qt.shape == x.t().shape
    same_codes(q, s, x)
    same_codes(qt, st, x.t())
    same_codes(*quantize_blocks(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_codes_of_any_strides_and_axes(dtype, path):
    x = features(40, 300, dtype)
    for view in (x[:, 1:258], x[::3, :200], x.t(), x[:, ::2], x[3:4], x[:1].expand(5, -1)):
        q, s, qt, st = quantize_blocks(view, transposed=True)
        same_codes(q, s, view)
        same_codes(qt, st, view.t())
    cube = x.view(5, 8, 300)
    q, s = quantize_blocks(cube)
    assert q.shape == (5, 8, 300) and s.shape == (5, 8, 3)
    same_codes(q.reshape(40, 300), s.reshape(40, 3), x)
    q, s = quantize_blocks(x[0])
    same_codes(q[None], s[None], x[:1])
    q, s, qt, st = quantize_blocks(x[:0], transposed=True)
    assert q.shape == (0, 300) and qt.shape == (300, 0) and st.shape == (300, 0)


def test_codes_at_the_types_borders(path):
    """Zeros, ties, maxima on a power of two's border, subnormal and largest
    values; a block with an infinity or a NaN is NaN, the others are not."""
    x = torch.zeros(12, 256, device=DEV)
    x[1, 3] = 448.0
    x[2, 3] = 448.0 * (1 + 2.0 ** -23)
    x[3] = torch.arange(256, device=DEV) / 16.0 - 3.0
    x[4, :5] = torch.tensor([1e-45, 2.0 ** -149, -1e-40, 2.0 ** -126, 3e-39], device=DEV)
    x[5] = torch.finfo(F32).max
    x[6, 0], x[6, 1] = 448.0, 464.0 / 2 ** 20
    x[7] = -2.0 ** -130
    x[8, :] = 1.0625 * 2.0 ** -7
    x[8, 7] = 1.0
    q, s, qt, st = quantize_blocks(x, transposed=True)
    same_codes(q, s, x)
    same_codes(qt, st, x.t())
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = torch.randn(200, 300, device=DEV)
        y[130, 129] = bad
        q, s, qt, st = quantize_blocks(y, transposed=True)
        assert s.view(torch.uint8)[130, 1] == 255 and (s.view(torch.uint8) == 255).sum() == 1
        assert q[130, 128:256].float().isnan().all() and q.float().isnan().sum() == 128
        assert st.view(torch.uint8)[129, 1] == 255 and (st.view(torch.uint8) == 255).sum() == 1
        assert qt[129, 128:].float().isnan().all() and qt.float().isnan().sum() == 72


def test_what_lies_behind_the_codes_stays():
    """Rows are padded to 16 codes; nothing past them is written."""
    x = features(5, 133, F32)
    q = torch.full((5, 160), 77, device=DEV, dtype=torch.uint8)
    s = torch.full((5, 8), 77, device=DEV, dtype=torch.uint8)
    L = _native.lib()
    assert L.cpab_b200_quantize_blocks(0, x.data_ptr(), 133, 5, 133, q.data_ptr(), 160, s.data_ptr(), 8, None, 0,
                                       None, 0, 0, None, None, None) == 0
    torch.cuda.synchronize()
    assert (q[:, 136:] == 77).all() and (s[:, 2:] == 77).all()
    same_codes(q[:, :133].view(CODES), s[:, :2].view(SCALES), x)


# ---- products --------------------------------------------------------------------

STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def near(y, x, w, bias, floor=0.0):
    """y against x w^T + bias of float64 values, element by element."""
    want = x @ w.t()
    size = x.abs() @ w.abs().t()
    off = (x.shape[1] / 32 + 4) * 2.0 ** -22 * size
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    off = off + 3 * 2.0 ** -24 * size
    off = off + STEP[y.dtype] * (want.abs() + off) + floor
    if y.dtype == F16:
        off = off + 2.0 ** -25
    assert y.shape == want.shape
    d = (y.double() - want).abs()
    assert (d <= off).all(), (d / off).max().item()


SIZES = [(1, 16, 16), (1, 4096, 128), (2, 40, 257), (16, 300, 1000), (8, 33, 3000), (9, 50, 127), (16, 20, 5000), (100, 64, 129), (128, 128, 128),
         (129, 65, 384), (257, 513, 640), (333, 1500, 1000), (515, 1003, 77), (1000, 260, 2049), (700, 1100, 1536)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", SIZES)
def test_products(size, dtype, path):
    M, N, K = size
    x, w = features(M, K, F32, 1), features(N, K, F32, 2) * K ** -0.5
    bias = torch.randn(N, device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    xq, ws = encoded(x), encoded(w)
    xv, wv = valued(*xq), valued(*ws)
    scale = 1.0 if dtype != F16 else 2.0 ** -6     # (half's range)
    q, s = quantize_blocks(x * scale)
    v, vs = quantize_blocks(w)
    near(matmul_quantized(q, s, v, vs, dtype=dtype), xv * scale, wv, None)
    near(matmul_quantized(q, s, v, vs, bias=bias.to(dtype), dtype=dtype), xv * scale, wv, bias.to(dtype))
    # float32 scales for rows, of either side
    rx = torch.rand(M, device=DEV) * scale + 0.1 * scale
    rw = torch.rand(N, device=DEV) + 0.1
    near(matmul_quantized(q, rx, v, rw, bias=bias, dtype=dtype), q.double() * rx.double()[:, None] * 1.0,
         v.double() * rw.double()[:, None], bias)
    near(matmul_quantized(q, rx, v, vs, dtype=dtype), q.double() * rx.double()[:, None], wv, None)


@pytest.mark.parametrize("size", [(2048, 2304, 256), (256, 20000, 128), (40000, 300, 384), (300, 300, 20000),
                                  (17, 361, 6942), (256, 128, 50001), (200, 70, 4097), (700, 650, 9000)])
def test_large_products(size, path):
    """Many tiles, tall, wide and long ones; the last rows and columns too."""
    M, N, K = size
    x, w = features(M, K, BF16, 4), features(N, K, BF16, 5)
    q, s = quantize_blocks(x)
    v, vs = quantize_blocks(w)
    y = matmul_quantized(q, s, v, vs)
    xv, wv = valued(*encoded(x)), valued(*encoded(w))
    near(y[-300:], xv[-300:], wv, None)
    near(y[:300], xv[:300], wv, None)


def test_long_sums_in_parts_with_scales_of_rows_and_bias(path):
    M, N, K = 40, 90, 9001
    x, w = features(M, K, F32, 6), features(N, K, F32, 7)
    b = torch.randn(N, device=DEV)
    q, _ = quantize_blocks(x)
    v, vs = quantize_blocks(w)
    r, u = torch.rand(M, device=DEV) + 0.1, torch.rand(N, device=DEV) + 0.1
    for dtype in (F32, BF16):
        near(matmul_quantized(q, r, v, u, bias=b, dtype=dtype), q.double() * r.double()[:, None],
             v.double() * u.double()[:, None], b)
        near(matmul_quantized(q, r, v, vs, bias=b, dtype=dtype), q.double() * r.double()[:, None],
             valued(*encoded(w)), b)


def test_product_of_every_block_of_scales():
    """A scale that belongs to another block, row or column would show: one code
    of 1 in one block of one row, its scale a power of its own."""
    for M, N, K in ((260, 300, 1500), (100, 60, 5000)):
        blocks_of_scales(M, N, K)


def blocks_of_scales(M, N, K):
    nb = -(-K // 128)
    s = (120 + torch.randint(0, 16, (M, nb), generator=torch.Generator().manual_seed(1))).to(DEV, torch.uint8)
    vs = (120 + torch.randint(0, 16, (N, nb), generator=torch.Generator().manual_seed(2))).to(DEV, torch.uint8)
    for b in (0, 3, 4, 7, 8, nb - 1):
        q = torch.zeros(M, K, device=DEV)
        q[:, b * 128 + 5] = 1.0
        q = quantize_blocks(q)[0].float().clamp_max(1.0).to(CODES)
        v = torch.zeros(N, K, device=DEV)
        v[:, b * 128 + 5] = 1.0
        v = v.to(CODES)
        y = matmul_quantized(q, s.view(SCALES), v, vs.view(SCALES), dtype=F32)
        want = torch.exp2(s[:, b].float() - 127)[:, None] * torch.exp2(vs[:, b].float() - 127)
        assert torch.equal(y, want)


def test_products_of_any_layout(path):
    """Codes off 16 bytes, scales with other strides, one row, leading axes."""
    M, N, K = 70, 90, 300
    x, w = features(M, K, F32, 6), features(N, K, F32, 7)
    xv, wv = valued(*encoded(x)), valued(*encoded(w))
    q, s = quantize_blocks(x)
    v, vs = quantize_blocks(w)
    want = matmul_quantized(q, s, v, vs, dtype=F32)
    near(want, xv, wv, None)
    loose = torch.zeros(M, K + 3, device=DEV, dtype=torch.uint8).view(CODES)[:, 3:]
    loose.copy_(q)
    turned = torch.empty(K, M, device=DEV, dtype=CODES).t()
    turned.copy_(q)
    ss = torch.empty(s.shape[1], M, device=DEV, dtype=torch.uint8).t()
    ss.copy_(s.view(torch.uint8))
    for a in (loose, turned, q.contiguous()):
        for b in (s, s.view(torch.uint8).contiguous().view(SCALES), ss.view(SCALES)):
            assert torch.equal(matmul_quantized(a, b, v, vs, dtype=F32), want)
            assert torch.equal(matmul_quantized(v, vs, a, b, dtype=F32).t(), want)
    # (few rows are summed in another order)
    one = matmul_quantized(q[3], s[3], v, vs, dtype=F32)
    near(one[None], xv[3:4], wv, None)
    assert torch.equal(matmul_quantized(q[3:4], s[3:4], v, vs, dtype=F32), one[None])
    assert torch.equal(matmul_quantized(loose[3:4], s[3:4].clone(), v, vs, dtype=F32), one[None])
    near(matmul_quantized(v[:, :K - 3], vs, q[:5, :K - 3].contiguous(), s[:5], dtype=F32).t(), xv[:5, :K - 3], wv[:, :K - 3], None)
    cube = matmul_quantized(q.view(7, 10, K), s.view(7, 10, -1), v, vs, dtype=F32)
    assert torch.equal(cube, want.view(7, 10, N))
    assert matmul_quantized(q[:0], s[:0], v, vs).shape == (0, N)
    assert matmul_quantized(q, s, v[:0], vs[:0]).shape == (M, 0)


@pytest.mark.parametrize("K", [1, 15, 19, 20, 35, 129, 1001, 4099])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_codes_whose_rows_begin_anywhere(rows, K, path):
    """From every offset in a word; the bytes before and behind are NaN codes."""
    x, w = features(rows, K, F32, 6), features(37, K, F32, 7)
    q, s = quantize_blocks(x)
    v, vs = quantize_blocks(w)
    want = matmul_quantized(q, s, v, vs, dtype=F32)
    for lead in range(5):
        loose = []
        for c in (q, v):
            t = torch.full((c.shape[0], K + 2 * lead + 1), 0x7F, device=DEV, dtype=torch.uint8).view(CODES)[:, lead:lead + K]
            loose.append(t.copy_(c))
        assert torch.equal(matmul_quantized(loose[0], s, loose[1], vs, dtype=F32), want)
        assert torch.equal(matmul_quantized(q, s, loose[1], vs, dtype=F32), want)
        assert torch.equal(matmul_quantized(loose[0], s, v, vs, dtype=F32), want)


def test_a_block_of_nan_reaches_its_row_alone(path):
    x, w = features(300, 500, F32, 8), features(200, 500, F32, 9)
    x[17, 130] = float("inf")
    y = matmul_quantized(*quantize_blocks(x), *quantize_blocks(w))
    assert y[17].isnan().all() and y.isnan().sum() == 200
    for rows in (slice(17, 18), slice(14, 20), slice(5, 18)):       # (few rows)
        y = matmul_quantized(*quantize_blocks(x[rows]), *quantize_blocks(w))
        assert y.isnan().sum() == 200 and y.isnan().all(1).sum() == 1
        y = matmul_quantized(*quantize_blocks(w), *quantize_blocks(x[rows]))
        assert y.isnan().sum() == 200 and y.isnan().all(0).sum() == 1
    # a NaN in the gradient reaches its row of dx, its column of the transposed product
    x[17, 130] = 0.0
    x.requires_grad_(True)
    dy = torch.ones(300, 200, device=DEV)
    dy[3, 7] = float("nan")
    (dx,) = torch.autograd.grad(linear_quantized(x, w), x, dy)
    assert dx[3].isnan().all() and dx.isnan().sum() == 500


def test_an_8_bit_norm_feeds_a_product(path):
    """rms_norm_quantized's rows against the weight's codes, bias in one rounding."""
    g = torch.Generator(DEV).manual_seed(0)
    x = torch.randn(33, 520, device=DEV, generator=g, dtype=F32)
    w = torch.randn(70, 520, device=DEV, generator=g)
    b = torch.randn(70, device=DEV, generator=g)
    q, scale = rms_norm_quantized(x, torch.ones(520, device=DEV))
    v, vs = quantize_blocks(w)
    near(matmul_quantized(q, scale, v, vs, bias=b, dtype=F32), q.double() * scale.double()[:, None],
         valued(*encoded(w)), b)


def test_products_on_another_stream_and_in_a_graph(path):
    x, w = features(200, 600, BF16, 10), features(300, 600, BF16, 11)
    want = matmul_quantized(*quantize_blocks(x), *quantize_blocks(w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = matmul_quantized(*quantize_blocks(x), *quantize_blocks(w))
    side.synchronize()
    assert torch.equal(got, want)
    a = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = matmul_quantized(*quantize_blocks(a), *quantize_blocks(w))
    for k in range(3):
        a.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, matmul_quantized(*quantize_blocks(a), *quantize_blocks(w)))


# ---- the trainable projection --------------------------------------------------------

TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (F16, F16, F16), (BF16, F32, F32), (BF16, BF16, F32)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("size", [(1, 16, 16), (5, 300, 129), (130, 48, 96), (515, 260, 1000), (1000, 700, 130)])
def test_projection_and_gradients(size, types, path):
    """As products of the codes of what each one sums."""
    M, N, K = size
    xt, wt, bt = types
    x, w = features(M, K, xt, 1, 0.5), (features(N, K, F32, 2, 0.3) * K ** -0.5).to(wt)
    b = torch.randn(N, device=DEV).to(bt)
    dy = features(M, N, xt, 3, 0.5)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear_quantized(x, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in leaves)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (xt, xt, wt, bt)
    v = lambda t: valued(*encoded(t.float()))  # noqa: E731
    near(y, v(x), v(w), b)
    near(dx, v(dy), v(w.t()).t().t(), None)
    near(dw, v(dy.t()), v(x.t()), None)
    size = dy.double().abs().sum(0)
    want = dy.double().sum(0)
    assert ((db.double() - want).abs() <= (M + 8) * 2.0 ** -24 * size + STEP[bt] * want.abs() + 2.0 ** -25).all()
    with torch.no_grad():
        assert torch.equal(linear_quantized(x, w, b), y)


def test_gradients_are_differences_of_exact_values(path):
    """Where all values are whole numbers that codes hold, the projection is
    exactly linear, and its gradients are its differences."""
    g = torch.Generator().manual_seed(0)
    M, N, K = 40, 24, 200
    whole = lambda *s: torch.randint(-7, 8, s, generator=g).float().to(DEV)  # noqa: E731
    x, w, b, dy = whole(M, K), whole(N, K), whole(N), whole(M, N)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear_quantized(*leaves), leaves, dy)
    f = lambda *a: (linear_quantized(*a).double() * dy.double()).sum()  # noqa: E731
    here = f(x, w, b)
    for _ in range(4):
        hx, hw, hb = whole(M, K), whole(N, K), whole(N)
        assert f(x + hx, w, b) - here == (dx.double() * hx.double()).sum()
        assert f(x, w + hw, b) - here == (dw.double() * hw.double()).sum()
        assert f(x, w, b + hb) - here == (db.double() * hb.double()).sum()


def test_gradients_only_where_asked(path):
    x, w, b = features(30, 40, F32), features(20, 40, F32), torch.zeros(20, device=DEV)
    dy = torch.randn(30, 20, device=DEV)
    full = torch.autograd.grad(linear_quantized(*[t.requires_grad_(True) for t in (x, w, b)]), (x, w, b), dy)
    for k in range(3):
        leaves = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(linear_quantized(*leaves), leaves[k], dy)[0], full[k])
    y = linear_quantized(x, w)
    assert torch.equal(torch.autograd.grad(y, (x, w), dy)[1], full[1])
    # the same leaf twice, a broadcast gradient, a batch of none
    s = torch.randn(16, 16, device=DEV).requires_grad_(True)
    linear_quantized(s, s).sum().backward()
    t = s.detach()
    ones = torch.ones(16, 16, device=DEV)
    v = lambda a: valued(*encoded(a))  # noqa: E731
    want = ones.double() @ v(t.t()).t() + ones.double() @ v(t.t()).t()
    assert (s.grad.double() - want).abs().max() <= 1e-5 * want.abs().max()
    e = x.detach()[:0].requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(linear_quantized(e, w, b).sum(), (e, w, b))
    assert gx.shape == (0, 40) and not gw.any() and not gb.any()


def test_leading_axes_and_once_only(path):
    x, w = features(24, 40, F32), features(20, 40, F32).requires_grad_(True)
    cube = x.view(2, 3, 4, 40).clone().requires_grad_(True)
    y = linear_quantized(cube, w)
    assert y.shape == (2, 3, 4, 20)
    flat = linear_quantized(x, w)
    assert torch.equal(y.view(24, 20), flat)
    dy = torch.randn(2, 3, 4, 20, device=DEV)
    assert torch.autograd.grad(y, cube, dy)[0].shape == cube.shape
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(linear_quantized(cube, w).sum(), cube, create_graph=True)
    with pytest.raises(RuntimeError, match="backward of linear_quantized|no gradient|forward|jvp|not implement"):
        with torch.autograd.forward_ad.dual_level():
            linear_quantized(torch.autograd.forward_ad.make_dual(x, x), w)


def test_a_training_step_in_a_graph(path):
    """Projection, gradients and all, captured; an eager graph of the same
    leaves is gone by then, as torch's capture asks for."""
    x = features(100, 64, BF16)
    w = (0.1 * torch.randn(48, 64, device=DEV)).to(BF16).requires_grad_(True)
    b = torch.zeros(48, device=DEV, dtype=BF16, requires_grad=True)
    dy = torch.randn(100, 48, device=DEV).to(BF16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(linear_quantized(x, w, b), (w, b), dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear_quantized(x, w, b)
        gw, gb = torch.autograd.grad(y, (w, b), dy)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(linear_quantized(x, w, b), (w, b), dy)
    assert torch.equal(gw, want[0]) and torch.equal(gb, want[1])


def test_results_are_the_same_from_run_to_run(path):
    x, w = features(2000, 900, BF16, 1), features(700, 900, BF16, 2).requires_grad_(True)
    b = torch.zeros(700, device=DEV, dtype=BF16, requires_grad=True)
    dy = features(2000, 700, BF16, 3)
    runs = [torch.autograd.grad(linear_quantized(x, w, b), (w, b), dy) for _ in range(3)]
    assert all(torch.equal(a, c) for r in runs[1:] for a, c in zip(runs[0], r))


def test_refusals(path):
    x, w = features(4, 32, F32), features(6, 32, F32)
    q, s = quantize_blocks(x)
    v, vs = quantize_blocks(w)
    with pytest.raises(TypeError, match="e4m3"):
        matmul_quantized(x, s, v, vs)
    with pytest.raises(TypeError, match="scale"):
        matmul_quantized(q, s.view(torch.uint8), v, vs)
    with pytest.raises(ValueError, match="scale"):
        matmul_quantized(q, s[:3], v, vs)
    with pytest.raises(ValueError, match="weight"):
        matmul_quantized(q, s, *quantize_blocks(w[:, :16]))
    with pytest.raises(TypeError, match="bias"):
        matmul_quantized(q, s, v, vs, bias=torch.zeros(6, device=DEV, dtype=F16))
    with pytest.raises(ValueError, match="bias"):
        matmul_quantized(q, s, v, vs, bias=torch.zeros(5, device=DEV))
    with pytest.raises(TypeError, match="dtype"):
        matmul_quantized(q, s, v, vs, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="scale"):
        matmul_quantized(q, s.cpu(), v, vs)
    with pytest.raises(RuntimeError, match="no gradient"):
        matmul_quantized(q, s, v, vs, bias=torch.zeros(6, device=DEV, requires_grad=True))
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_blocks(x.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="weight"):
        linear_quantized(x, w[:, :16])
    with pytest.raises(TypeError, match="weight"):
        linear_quantized(x, w.to(BF16))
    with pytest.raises(ValueError, match="transpose"):
        quantize_blocks(x[None], transposed=True)


def test_a_vector_through_a_projection(path):
    x, w, b = features(1, 200, F32)[0].requires_grad_(True), features(30, 200, F32, 1).requires_grad_(True), torch.zeros(30, device=DEV)
    y = linear_quantized(x, w, b)
    assert y.shape == (30,)
    dy = torch.randn(30, device=DEV)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    v = lambda t: valued(*encoded(t.detach()))  # noqa: E731
    near(y[None], v(x[None]), v(w), None)
    near(dx[None], v(dy[None]), v(w.t()), None)
    near(dw, v(dy[:, None]), v(x[None].t()), None)


def test_two_streams_at_once(path):
    """Calls that overlap share nothing."""
    xs = [features(700, 900, BF16, k) for k in range(4)]
    w = features(800, 900, BF16, 9)
    want = [linear_quantized(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(5):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(linear_quantized(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
