"""Host-side checks of the 8-bit projections and the orthogonalised steps: the
C ABI's refusals, the Python layer's argument errors (no GPU needed)."""
import ctypes

import pytest
import torch

from cpab import _ext, _native
from cpab.optim import Muon, muon_, orthogonalize
from cpab.pytorch.localizer import SeriesLocalizer
from cpab.pytorch.projection import linear_quantized, matmul_quantized, quantize_blocks

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
OFF = ctypes.c_void_p(4100)


def err():
    return _native.lib().cpab_b200_last_error().decode()


def call(fn, base, **kw):
    a = list(base)
    for i, v in kw.items():
        a[int(i[1:])] = v
    return fn(*a)


def test_quantize_entry_point_validates():
    L = _native.lib()
    # dtype, x, row, rows, columns, q, row, scale, row, qt, row, scale_t, row, sum dtype, sum, workspace, stream
    ok = [2, P, 200, 40, 200, P, 208, P, 4, P, 48, P, 4, 0, P, P, None]
    f = L.cpab_b200_quantize_blocks
    assert call(f, ok, a0=3) == -1 and "type" in err()
    assert call(f, ok, a13=3) == -1
    assert call(f, ok, a3=-1) == -1 and "negative" in err()
    assert call(f, ok, a3=1 << 31) == -4
    assert call(f, ok, a1=None) == -1 and "null" in err()
    assert call(f, ok, a5=OFF) == -1 and "16" in err()
    assert call(f, ok, a6=200) == -1 and call(f, ok, a6=192) == -1 and call(f, ok, a8=1) == -1
    assert call(f, ok, a7=None) == -1
    assert call(f, ok, a9=OFF) == -1 and call(f, ok, a10=32) == -1 and call(f, ok, a12=0) == -1
    assert call(f, ok, a15=None) == -1 and "workspace" in err()
    assert call(f, ok, a5=None, a9=None, a14=None) == -1 and "nothing" in err()
    assert call(f, ok, a3=0, a14=None) == 0 and err() == ""
    assert L.cpab_b200_quantize_blocks_workspace(129, 7) == 14
    assert L.cpab_b200_quantize_blocks_workspace(-1, 7) == 0


def test_product_entry_point_validates():
    L = _native.lib()

    def operand(codes=4096, row=208, scale=4096, scale_row=4):
        return _native._Quantized(codes, row, scale, scale_row)

    def one(x=None, w=None, dtype=0, M=8, N=8, K=200, bias_dtype=0, bias=None, y=P, y_row=8):
        x, w = x or operand(), w or operand()
        return L.cpab_b200_matmul_quantized(dtype, ctypes.byref(x), ctypes.byref(w), M, N, K, bias_dtype, bias, y,
                                            y_row, P, None)

    assert one(dtype=4) == -1 and "type" in err()
    assert one(dtype=2, bias_dtype=1, bias=P) == -1 and "bias" in err()
    assert one(M=-1) == -1 and one(K=0) == -1 and one(y_row=7) == -1
    assert one(M=1 << 31) == -4
    assert one(y=None) == -1 and "null" in err()
    assert one(x=operand(codes=None)) == -1 and one(w=operand(scale=None)) == -1 and "null" in err()
    assert one(x=operand(codes=4104)) == -1 and "16" in err()
    assert one(x=operand(row=200)) == -1 and one(x=operand(row=192)) == -1
    assert one(w=operand(scale_row=1)) == -1 and "scales" in err()
    assert one(w=operand(scale=4098, scale_row=0)) == -1 and "float32" in err()
    assert one(M=0) == 0 and one(N=0) == 0 and err() == ""
    assert L.cpab_b200_matmul_quantized(0, None, None, 8, 8, 8, 0, None, P, 8, None, None) == -1
    w = L.cpab_b200_matmul_quantized_workspace
    assert w(0, 8, 8) == 0 and w(8, 8, 0) == 0 and w(4096, 4096, 512) == 0


def test_layout_entry_point_validates():
    L = _native.lib()
    one = lambda v: (ctypes.c_void_p * 1)(v)  # noqa: E731
    size = lambda v: (ctypes.c_int64 * 1)(v)  # noqa: E731
    ok = [1, one(4097), size(33), size(5), one(4096), 33, None]
    f = L.cpab_b200_lay_out_codes
    assert call(f, ok, a0=3) == -1 and call(f, ok, a5=0) == -1 and call(f, ok, a1=None) == -1
    assert call(f, ok, a4=one(4100)) == -1 and "16" in err()
    assert call(f, ok, a1=one(None)) == -1 and call(f, ok, a3=size(-1)) == -1
    assert call(f, ok, a3=size(1 << 31)) == -4
    assert call(f, ok, a3=size(0)) == 0 and call(f, ok, a0=0) == 0 and err() == ""


COEFFICIENTS = (ctypes.c_double * 3)(3.4445, -4.775, 2.0315)


def test_orthogonalize_entry_point_validates():
    L = _native.lib()
    # dtype, x, batch, rows, columns, steps, coefficients, eps, out, workspace, stream
    ok = [2, P, 1, 300, 400, 5, COEFFICIENTS, 1e-7, P, P, None]
    f = L.cpab_b200_orthogonalize
    assert call(f, ok, a0=-1) == -1 and "type" in err()
    assert call(f, ok, a2=-1) == -1 and call(f, ok, a6=None) == -1
    assert call(f, ok, a5=0) == -1 and call(f, ok, a5=65) == -1 and "steps" in err()
    assert call(f, ok, a7=-1.0) == -1 and call(f, ok, a7=float("nan")) == -1 and "eps" in err()
    for c in ((100.0, 0.0, 0.0), (3.0, -61.0, 0.0), (float("nan"), 0.0, 0.0), (3.0, float("inf"), 1.0)):
        assert call(f, ok, a6=(ctypes.c_double * 3)(*c)) == -1 and "outgrow" in err()
    assert call(f, ok, a3=(1 << 20) + 1) == -4 and call(f, ok, a2=65537) == -4
    assert call(f, ok, a1=None) == -1 and call(f, ok, a8=None) == -1 and call(f, ok, a9=OFF) == -1
    assert call(f, ok, a2=0) == 0 and call(f, ok, a4=0) == 0 and err() == ""
    w = L.cpab_b200_orthogonalize_workspace
    assert w(2, 1, 300, 400) > 0 and w(2, 1, 130, 260) > 0 and w(2, 1, 64, 260) == 0 and w(7, 1, 8, 8) == 0 and w(2, 0, 8, 8) == 0 and w(2, 1, 8, (1 << 20) + 1) == 0


def test_muon_entry_point_validates():
    L = _native.lib()
    t = (_native._MuonTensor * 1)()

    def one(count=1, coefficients=COEFFICIENTS, steps=5, eps=1e-7, adjust=0, work=P, **kw):
        base = dict(param=4096, grad=4096, momentum=8192, rows=300, columns=400, dtype=0)
        for k, v in {**base, **kw}.items():
            setattr(t[0], k, v)
        return L.cpab_b200_muon(ctypes.byref(t), count, 0.1, None, 0.9, 1, 0.1, steps, coefficients, eps, adjust, work,
                                None)

    assert one(dtype=5) == -1 and "type" in err()
    assert one(rows=-1) == -1 and one(columns=(1 << 20) + 1) == -1 and "size" in err()
    for k in ("param", "grad", "momentum"):
        assert one(**{k: None}) == -1 and "null" in err()
    assert one(steps=0) == -1 and one(eps=-1.0) == -1 and one(adjust=2) == -1 and one(count=-1) == -1
    assert one(coefficients=None) == -1
    assert one(work=None) == -1 and one(work=OFF) == -1 and "workspace" in err()
    assert one(rows=0, work=None) == 0 and err() == ""
    assert L.cpab_b200_muon(None, 1, 0.1, None, 0.9, 1, 0.1, 5, COEFFICIENTS, 1e-7, 0, P, None) == -1
    one()
    two = (_native._MuonTensor * 2)(t[0], t[0])
    two[1].momentum = 16384
    assert L.cpab_b200_muon(ctypes.byref(two), 2, 0.1, None, 0.9, 1, 0.1, 5, COEFFICIENTS, 1e-7, 0, P, None) == -1
    assert "twice" in err()
    assert L.cpab_b200_muon_workspace(ctypes.byref(t), 1) > 0
    assert L.cpab_b200_muon_workspace(None, 1) == 0


@pytest.fixture(params=["ext", "python"])
def path(request):
    if request.param == "python":
        with _ext.python_path():
            yield
    else:
        assert _ext.module() is not None
        yield


def test_cpu_tensors_are_refused(path):
    x, w = torch.randn(4, 32), torch.randn(8, 32)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_blocks(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        matmul_quantized(q, s, q, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_quantized(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        orthogonalize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        muon_([x], [x], [x], lr=0.1)


def test_gradients_are_refused(path):
    x = torch.randn(4, 32, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize_blocks(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        orthogonalize(x)


def test_options_are_checked():
    p = [torch.nn.Parameter(torch.zeros(3, 4))]
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(eps=-1e-8), dict(ns_steps=0),
                dict(adjust_lr_fn="other"), dict(ns_coefficients=(1.0, 2.0))):
        with pytest.raises(ValueError):
            Muon(p, **bad)
    with pytest.raises(ValueError, match="matrices"):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    opt = Muon(p)
    opt.step()                                         # no gradients: nothing to do
    assert not opt.state.get(p[0])
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(3, 4, 5))]})
    assert len(opt.param_groups) == 1
    q = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="adjust_lr"):
        muon_([q], [q], [q], lr=0.1, adjust_lr="other")
    with pytest.raises(ValueError, match="lr"):
        muon_([q], [q], [q], lr=torch.tensor(0.1))
    with pytest.raises(ValueError, match="projection_bits"):
        SeriesLocalizer(1, 3, projection_bits=4)


def test_other_devices_are_refused(path):
    """Before anything is launched (tensors without memory, so no GPU is needed)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    native = _native if _ext.module() is None else _ext.module()
    with FakeTensorMode():
        a, b = (torch.empty(4, 32, device="cuda:%d" % k) for k in (0, 1))
        q, s = torch.empty(4, 32, device="cuda:0", dtype=torch.float8_e4m3fn), torch.empty(4, device="cuda:1")
        with pytest.raises(RuntimeError, match="cuda:1"):
            native.matmul_quantized(q, s, q, s, None, torch.bfloat16)
        with pytest.raises(RuntimeError, match="cuda:1"):
            linear_quantized(a, b)
        with pytest.raises(RuntimeError, match="device"):
            native.muon([a], [b], [a], 0.1, None, 0.9, True, 0.1, 5, (3.0, -4.0, 2.0), 1e-7, 0)
        with pytest.raises(RuntimeError, match="device"):
            native.muon([a], [a], [a], 0.0, torch.empty(1, device="cuda:1"), 0.9, True, 0.1, 5, (3.0, -4.0, 2.0),
                        1e-7, 0)
