"""quantize_blocks, matmul_quantized and linear_quantized at the edges of what
they take."""
import contextlib
import ctypes

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.projection import linear_quantized, matmul_quantized, quantize_blocks
from test_gpu_projection import near, valued

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


@pytest.fixture(params=["ext", "python"])
def path(request):
    with _ext.python_path() if request.param == "python" else contextlib.nullcontext():
        yield request.param


@pytest.mark.parametrize("M", [1, 9, 16, 40, 200])
def test_codes_made_anew_in_one_buffer(M):
    """Codes of one input after another in the same place, each followed by its
    product, in a chain of launches that begin while the one before runs: every
    product is that of its own codes.  Captured, and replayed with other inputs."""
    K, N, rounds = 640, 96, 6
    L = _native.lib()
    g = torch.Generator().manual_seed(M)
    w, ws = quantize_blocks(torch.randn(N, K, generator=g).to(DEV))
    xs = torch.empty(rounds, M, K, device=DEV)
    q, s = torch.empty(M, K, device=DEV, dtype=torch.uint8), torch.empty(M, 8, device=DEV, dtype=torch.uint8)
    ys = torch.empty(rounds, M, N, device=DEV)
    x_op = _native._Quantized(q.data_ptr(), K, s.data_ptr(), 8)
    w_op = _native._Quantized(w.data_ptr(), w.stride(0), ws.data_ptr(), ws.stride(0))
    floats = L.cpab_b200_matmul_quantized_workspace(M, N, K)
    work = torch.empty(max(floats, 8), device=DEV)

    def chain():
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        for k in range(rounds):
            assert L.cpab_b200_quantize_blocks(0, xs[k].data_ptr(), K, M, K, q.data_ptr(), K, s.data_ptr(), 8, None, 0,
                                               None, 0, 0, None, None, stream) == 0
            assert L.cpab_b200_matmul_quantized(0, ctypes.byref(x_op), ctypes.byref(w_op), M, N, K, 0, None,
                                                ys[k].data_ptr(), N, work.data_ptr(), stream) == 0

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for turn in range(30):
        xs.copy_(torch.randn(rounds, M, K, generator=g))
        ys.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for k in range(rounds):
            one = quantize_blocks(xs[k])
            torch.cuda.synchronize()
            assert torch.equal(ys[k], matmul_quantized(*one, w, ws, dtype=F32)), (turn, k)


# Rows that take each of the kernels: one pass (8 and 16 rows at a time), tiles, tiles
# whose sum is cut into parts, pairs of tiles.
ROWS = [(1, 70, 300), (8, 70, 300), (9, 70, 300), (16, 70, 300), (17, 70, 300), (40, 90, 9001), (300, 200, 500)]


def codes(R, K, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, K, generator=g) * 20).to(DEV).to(CODES)


def powers(R, K, near_, seed):
    """Scales of blocks, as bytes, within 8 times of 2^near_."""
    g = torch.Generator().manual_seed(seed)
    return (127 + near_ + torch.randint(-3, 4, (R, -(-K // 128)), generator=g)).to(torch.uint8).to(DEV)


def by_blocks(q, s):
    return valued(q, s.long() - 127)


def by_rows(q, r):
    return q.double() * r.double()[:, None]


@pytest.mark.parametrize("far", [(115, -108), (-108, 115), (-120, 110), (124, -124)])
@pytest.mark.parametrize("size", ROWS)
def test_scales_of_blocks_far_apart(size, far, path):
    """One scale near float32's end, the other near its beginning: the result is
    neither, whichever kernel the number of rows takes."""
    M, N, K = size
    q, v = codes(M, K, 1), codes(N, K, 2)
    s, vs = powers(M, K, far[0], 3), powers(N, K, far[1], 4)
    y = matmul_quantized(q, s.view(SCALES), v, vs.view(SCALES), dtype=F32)
    near(y, by_blocks(q, s), by_blocks(v, vs), None)
    if M > 1:                       # a row alone is what it is among others
        one = matmul_quantized(q[:1], s[:1].view(SCALES), v, vs.view(SCALES), dtype=F32)
        near(one, by_blocks(q[:1], s[:1]), by_blocks(v, vs), None)


@pytest.mark.parametrize("far", [(1e30, 1e-33), (1e-37, 1e36), (3e38, 1e-38), (1e-44, 1e38)])
@pytest.mark.parametrize("size", ROWS)
def test_scales_of_rows_far_apart(size, far, path):
    M, N, K = size
    q, v = codes(M, K, 1), codes(N, K, 2)
    g = torch.Generator().manual_seed(5)
    r, u = (((0.5 + torch.rand(n, generator=g) / 2) * f).to(DEV) for n, f in zip((M, N), far))
    b = torch.randn(N, generator=g).to(DEV) * (far[0] * far[1])
    for bias in (None, b):
        near(matmul_quantized(q, r, v, u, bias=bias, dtype=F32), by_rows(q, r), by_rows(v, u), bias)


@pytest.mark.parametrize("far", [(1e-33, 110), (1e30, -105), (2e-38, 124), (1e-44, 119)])
@pytest.mark.parametrize("size", ROWS)
def test_a_scale_of_rows_far_from_those_of_blocks(size, far, path):
    M, N, K = size
    g = torch.Generator().manual_seed(6)
    for rows_first in (True, False):
        q, v = codes(M, K, 1), codes(N, K, 2)
        R, B = (M, N) if rows_first else (N, M)
        r = ((0.5 + torch.rand(R, generator=g) / 2) * far[0]).to(DEV)
        s = powers(B, K, far[1], 7)
        if rows_first:
            y, x, w = matmul_quantized(q, r, v, s.view(SCALES), dtype=F32), by_rows(q, r), by_blocks(v, s)
        else:
            y, x, w = matmul_quantized(q, s.view(SCALES), v, r, dtype=F32), by_blocks(q, s), by_rows(v, r)
        near(y, x, w, None)


def test_scales_of_nothing_and_of_no_number(path):
    """A row's scale of 0, an infinity or a NaN is what it is beside any other's."""
    q, v = codes(20, 200, 1), codes(30, 200, 2)
    u = torch.full((30,), 1e-30, device=DEV)
    s = powers(30, 200, -100, 3)
    r = torch.ones(20, device=DEV)
    r[3], r[5], r[7], r[9] = 0.0, float("inf"), float("nan"), -2e30
    for rows in (slice(0, 20), slice(0, 10), slice(3, 4), slice(5, 6)):
        for scale, value in ((u, by_rows(v, u)), (s.view(SCALES), by_blocks(v, s))):
            y = matmul_quantized(q[rows], r[rows], v, scale, dtype=F32)
            want = (q[rows].double() @ value.t()) * r[rows].double()[:, None]
            assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf())
            ok = want.isfinite()
            assert (y.double() - want)[ok].abs().max() <= 1e-5 * want[ok].abs().max() if ok.any() else True
            assert torch.equal(y[want.isinf()].sign(), want[want.isinf()].sign().float())


def drift(M, N, K, dtype):
    """The mean relative error of sums of like signs, of 16 x 64 results (rows of other
    sizes, so that their roundings differ)."""
    g = torch.Generator(DEV).manual_seed(1)
    # codes of 2^-5 to 3.75, whose products are multiples of 2^-16
    q, v = (torch.randint(0x10, 0x48, (n, K), device=DEV, dtype=torch.uint8, generator=g).view(CODES) for n in (M, N))
    r, u = (torch.rand(n, device=DEV, generator=g) * f + f for n, f in ((M, 1.0), (N, 2.0 ** -30)))
    y = matmul_quantized(q, r, v, u, dtype=dtype)
    rows, columns = torch.arange(0, M, max(1, M // 16)), torch.arange(0, N, max(1, N // 64))
    want = sum(q[rows, k:k + 32768].double() @ v[columns, k:k + 32768].double().t() for k in range(0, K, 32768))
    want = want * r[rows].double()[:, None] * u[columns].double()
    return ((y[rows][:, columns].double() - want) / want).mean().item()


@pytest.mark.parametrize("size", [(2048, 2048, 32768), (2048, 2048, 131072), (1000, 1000, 65536), (128, 2048, 65536),
                                  (64, 64, 262144)])
def test_long_sums_of_like_signs_do_not_drift(size):
    """What an instruction of 32 codes cuts off its sum is less than 2^-23 of it and has
    one sign, evenly spread.  A sum that grows evenly is cut, in the mean over its course,
    by half of half of that: n instructions' errors come to n / 4 2^-23 of it (the sum is
    at a power of two's end at worst).  Float32 sums begin anew every 256 instructions,
    and are then added with roundings, which have both signs."""
    assert abs(drift(*size, F32)) <= (256 + 1) / 4 * 2.0 ** -23 + 2.0 ** -24


def test_very_long_sums_of_like_signs_do_not_drift_in_16_bits():
    """As above with 512 instructions; a rounding to bfloat16, 2^-8 at most, has both
    signs: the mean of 1024 of them is within 5 sqrt(1 / 3 / 1024) 2^-8."""
    assert abs(drift(1600, 1600, 1 << 20, BF16)) <= (512 + 1) / 4 * 2.0 ** -23 + 5 * (1 / 3 / 1024) ** 0.5 * 2.0 ** -8


def test_a_product_refuses_forward_derivatives_of_its_scales(path):
    q, s = codes(4, 32, 1), torch.ones(4, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(s, s)
        for args in ((q, dual, q, s), (q, s, q, dual)):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                matmul_quantized(*args)


@pytest.mark.parametrize("lead", [(5,), (2, 3), (), (0,)])
def test_a_projection_without_outputs(lead, path):
    """A weight of no rows: a gradient of zeros for x, empty ones for the others."""
    x = torch.randn(*lead, 40, device=DEV, requires_grad=True)
    w, b = (torch.empty(s, device=DEV, requires_grad=True) for s in ((0, 40), (0,)))
    for bias in (None, b):
        y = linear_quantized(x, w, bias)
        assert y.shape == (*lead, 0)
        leaves = [x, w] + ([b] if bias is not None else [])
        dx, *others = torch.autograd.grad(y.sum(), leaves)
        assert dx.shape == x.shape and not dx.any()
        assert [g.shape for g in others] == [t.shape for t in leaves[1:]]
    (gw,) = torch.autograd.grad(linear_quantized(x.detach(), w).sum(), w)
    assert gw.shape == (0, 40)
