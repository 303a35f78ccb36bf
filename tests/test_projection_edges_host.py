"""Host-side checks at the edges of the 8-bit projections and the orthogonalised
steps (no GPU needed)."""
import ctypes
import os
import re

import pytest
import torch

from cpab import _ext, _native
from cpab.pytorch.projection import matmul_quantized

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fg-cpab_b200", "csrc")


def code_of(name):
    """A source file without its comments."""
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name", sorted(n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh"))))
def test_kernels_that_begin_early_read_with_ordinary_loads(name):
    """A kernel that waits for the one before (griddepcontrol.wait) runs while that
    one writes: read-only loads may return what was there before."""
    code = code_of(name)
    if not re.search(r"griddepcontrol\.wait|\bdep_wait\b", code):
        pytest.skip("no kernel of this file begins early")
    assert not re.findall(r"__ldg|ld\.global(?:\.\w+)*\.nc|__restrict__", code)


@pytest.fixture(params=["ext", "python"])
def path(request):
    if request.param == "python":
        with _ext.python_path():
            yield
    else:
        assert _ext.module() is not None
        yield


def test_a_product_refuses_scales_and_codes_that_want_a_gradient(path):
    """A row's float32 scale is an ordinary tensor of a graph: its gradient would be lost."""
    q, s = torch.zeros(4, 32).to(torch.float8_e4m3fn), torch.ones(4)
    wanting = torch.ones(4, requires_grad=True)
    for args in ((q, wanting, q, s), (q, s, q, wanting), (q, wanting * 2, q, s),
                 (q.clone().requires_grad_(True), s, q, s), (q, s, q.clone().requires_grad_(True), s)):
        with pytest.raises(RuntimeError, match="no gradient"):
            matmul_quantized(*args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            matmul_quantized(*args)
    with pytest.raises(RuntimeError, match="no gradient"):
        matmul_quantized(q, s, q, s, bias=wanting)


def test_a_wait_limit_is_a_time():
    L = _native.lib()
    assert L.cpab_b200_set_wait_limit(-1) == -1 and b"negative" in L.cpab_b200_last_error()
    assert L.cpab_b200_set_wait_limit(0) == 0 and L.cpab_b200_set_wait_limit(2 * 10 ** 9) == 0


def test_muon_refuses_a_gradient_that_is_a_momentum():
    """The momentum is written before the gradient is read the second time."""
    L = _native.lib()
    coefficients = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)
    for rows in (300, 20):
        for grads in ((8192, 4096), (4096, 65536), (65536, 8192)):
            t = (_native._MuonTensor * 2)()
            for k in range(2):
                t[k] = _native._MuonTensor(1 << 20 << k, grads[k], (8192, 65536)[k], rows, 20, 0)
            assert L.cpab_b200_muon(ctypes.byref(t), 2, 0.1, None, 0.9, 1, 0.1, 5, coefficients, 1e-7, 0,
                                    ctypes.c_void_p(4096), None) == -1
            assert b"momentum" in L.cpab_b200_last_error()
