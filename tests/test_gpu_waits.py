"""Waits inside the product kernels that run out: the call's results are NaN, the
kernels return, and the next call says so.  (With a limit of 0 the roles of a block
give up before they hand one another anything, so nothing is left to wait for.)"""
import contextlib
import os
import subprocess
import sys

import pytest
import torch

from cpab import _ext, _native
from cpab.optim import muon_, orthogonalize
from cpab.pytorch.projection import linear_quantized, matmul_quantized, quantize_blocks

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
DEFAULT = 2 * 10 ** 9


@pytest.fixture(params=["ext", "python"])
def path(request):
    with _ext.python_path() if request.param == "python" else contextlib.nullcontext():
        yield request.param


@contextlib.contextmanager
def no_waiting():
    L = _native.lib()
    assert L.cpab_b200_set_wait_limit(0) == 0
    try:
        yield
    finally:
        assert L.cpab_b200_set_wait_limit(DEFAULT) == 0
        torch.cuda.synchronize()


def reported(call):
    """The next call raises, once; the one after it answers."""
    with pytest.raises(RuntimeError, match="gave up waiting"):
        call()
    return call()


# 128 x 64 and 128 x 128 tiles, pairs, sums in parts, in segments
@pytest.mark.parametrize("size", [(40, 64, 129), (1024, 1024, 1024), (2048, 2304, 256), (256, 128, 50001),
                                  (2048, 2048, 20000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_products(size, dtype, path):
    M, N, K = size
    g = torch.Generator(DEV).manual_seed(0)
    x = quantize_blocks(torch.randn(M, K, device=DEV, generator=g))
    w = quantize_blocks(torch.randn(N, K, device=DEV, generator=g))
    call = lambda: matmul_quantized(*x, *w, dtype=dtype)  # noqa: E731
    want = call()
    with no_waiting():
        y = call()
    assert y.isnan().all()
    assert torch.equal(reported(call), want)


@pytest.mark.parametrize("shape", [(130, 260), (3, 300, 500), (1100, 1300), (256, 4096)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_orthogonalisations(shape, dtype, path):
    x = torch.randn(shape, device=DEV, generator=torch.Generator(DEV).manual_seed(0)).to(dtype)
    call = lambda: orthogonalize(x)  # noqa: E731
    want = call()
    with no_waiting():
        y = call()
    assert y.isnan().all()
    assert torch.equal(reported(call), want)


def test_a_step_is_not_taken_after_one(path):
    """The call that reports leaves parameters and momenta as they are; calls whose
    kernels do not wait report too, and their own results never depend on the limit."""
    x = torch.randn(130, 260, device=DEV)
    p, m = torch.randn(140, 200, device=DEV), torch.zeros(140, 200, device=DEV)
    g = torch.randn(140, 200, device=DEV)
    with no_waiting():
        orthogonalize(x)
    before = p.clone()
    with pytest.raises(RuntimeError, match="gave up waiting"):
        muon_([p], [g], [m], lr=0.1)
    assert torch.equal(p, before) and not m.any()
    muon_([p], [g], [m], lr=0.1)
    assert p.isfinite().all() and not torch.equal(p, before)
    a, b = quantize_blocks(x[:5]), quantize_blocks(x)
    want = matmul_quantized(*a, *b)
    with no_waiting():
        assert torch.equal(matmul_quantized(*a, *b), want)
        small = orthogonalize(x[:60, :70])
    assert torch.equal(orthogonalize(x[:60, :70]), small)
    with no_waiting():
        y = linear_quantized(x, x)
    assert y.isnan().all()
    with pytest.raises(RuntimeError, match="gave up waiting"):
        linear_quantized(x, x)
    assert linear_quantized(x, x).isfinite().all()


def test_captured_products_report_to_the_next_call():
    """The limit is a launch's: a captured one keeps its own."""
    x = torch.randn(300, 500, device=DEV)
    want = orthogonalize(x)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orthogonalize(x)
    with no_waiting():
        with torch.cuda.graph(other):
            z = orthogonalize(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(orthogonalize(x), want)
    other.replay()
    torch.cuda.synchronize()
    assert z.isnan().all()
    assert torch.equal(reported(lambda: orthogonalize(x)), want)


FIRST = """
import torch
from cpab.optim import orthogonalize
from cpab.pytorch.projection import matmul_quantized, quantize_blocks
x = torch.randn(300, 500, device="cuda")
q = quantize_blocks(x)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, z = matmul_quantized(*q, *q), orthogonalize(x)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, matmul_quantized(*q, *q)) and torch.equal(z, orthogonalize(x))
print("captured")
"""


def test_the_first_product_of_a_process_is_captured():
    """What is set up at a device's first product may be set up in a capture."""
    env = {**os.environ, "PYTHONPATH": os.pathsep.join(p for p in sys.path if p)}
    run = subprocess.run([sys.executable, "-c", FIRST], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr[-2000:]
