"""quantize_blocks, matmul_quantized and linear_quantized at the edges of what
they take."""
import contextlib
import ctypes

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.projection import matmul_quantized, quantize_blocks

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
