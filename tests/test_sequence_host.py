"""Host-side checks of the sequence-network operators: the C ABI's refusals,
the Python layer's argument errors (no GPU needed)."""
import ctypes

import pytest
import torch

from cpab import _ext, _native
from cpab.optim import AdamW, adamw_
from cpab.pytorch.norm import rms_norm, rms_norm_quantized
from cpab.pytorch.recurrence import gated_scan, gated_scan_step

P = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def err():
    return _native.lib().cpab_b200_last_error().decode()


def call(fn, base, **kw):
    a = list(base)
    for i, v in kw.items():
        a[int(i[1:])] = v
    return fn(*a)


def test_scan_entry_points_validate():
    L = _native.lib()
    # dtype, x, strides, gate, strides, B, T, D, lengths, h0, h, last, states, workspace, stream
    ok = [2, P, 64, 8, P, 64, 8, 2, 8, 8, None, None, P, P, P, P, None]
    f = L.cpab_b200_gated_scan
    assert call(f, ok, a0=3) == -1 and "dtype" in err()
    assert call(f, ok, a1=None) == -1 and "null" in err()
    assert call(f, ok, a4=None) == -1
    assert call(f, ok, a7=-1) == -1 and "negative" in err()
    assert call(f, ok, a8=1 << 31) == -4 and "2^31" in err()
    assert call(f, ok, a7=1 << 20, a9=1 << 11) == -4 and "2^30" in err()
    assert call(f, ok, a12=None) == -1 and "output" in err()
    assert call(f, ok, a15=None) == -1 and "workspace" in err()
    assert call(f, ok, a15=ctypes.c_void_p(4100)) == -1
    assert call(f, ok, a7=0) == 0 and err() == ""
    assert call(f, ok, a8=0, a13=None) == 0            # no samples, no state wanted
    # ..., lengths, states, grad_h, grad_last, grad_x, strides, grad_gate, strides, grad_h0, workspace,
    # stream
    okb = [2, P, 64, 8, P, 64, 8, 2, 8, 8, None, P, P, P, P, 64, 8, P, 64, 8, P, P, None]
    g = L.cpab_b200_gated_scan_backward
    assert call(g, okb, a11=None) == -1 and "states" in err()
    assert call(g, okb, a14=None) == -1 and call(g, okb, a17=None) == -1
    assert call(g, okb, a0=-1) == -1
    assert call(g, okb, a21=None) == -1 and "workspace" in err()
    assert call(g, okb, a9=0) == 0
    # dtype, x, row, gate, row, B, D, slots, rows, state, h, stream
    oks = [0, P, 8, P, 8, 2, 8, None, 2, P, P, None]
    s = L.cpab_b200_gated_scan_step
    assert call(s, oks, a8=1) == -1 and "state rows" in err()
    assert call(s, oks, a9=None) == -1 and call(s, oks, a10=None) == -1
    assert call(s, oks, a5=0) == 0
    assert L.cpab_b200_gated_scan_chunk() > 0
    assert L.cpab_b200_gated_scan_workspace(2, 3, 100, 64) > 0
    assert L.cpab_b200_gated_scan_workspace(2, 3, 1 << 31, 64) == 0


def test_norm_entry_points_validate():
    L = _native.lib()
    # dtype, stream, weight, x, row, residual, row, w, rows, D, eps, y, sum, rstd, stream
    ok = [2, 2, 0, P, 8, P, 8, P, 4, 8, 1e-6, P, P, P, None]
    f = L.cpab_b200_rms_norm
    assert call(f, ok, a0=7) == -1 and "types" in err()
    assert call(f, ok, a1=1) == -1 and call(f, ok, a2=1) == -1
    assert call(f, ok, a9=0) == -1 and "shape" in err()
    assert call(f, ok, a9=16385) == -4 and "16384" in err()
    assert call(f, ok, a10=-1.0) == -1 and "eps" in err()
    assert call(f, ok, a10=float("nan")) == -1
    assert call(f, ok, a12=None) == -1 and "null" in err()
    assert call(f, ok, a8=1 << 31) == -4
    assert call(f, ok, a8=0) == 0 and err() == ""
    # ..., eps, q, scale, sum, stream
    okq = [2, 2, 0, P, 8, P, 8, P, 4, 8, 1e-6, P, P, P, None]
    q = L.cpab_b200_rms_norm_quantized
    assert call(q, okq, a11=None) == -1 and call(q, okq, a12=None) == -1
    assert call(q, okq, a13=None) == -1 and call(q, okq, a9=-3) == -1
    # dtype, stream, weight, sum, row, w, rstd, rows, D, gy, gs, gx, gres, work, gw, stream
    okb = [2, 2, 0, P, 8, P, P, 4, 8, P, P, P, None, P, P, None]
    b = L.cpab_b200_rms_norm_backward
    assert call(b, okb, a13=None) == -1 and "workspace" in err()
    assert call(b, okb, a12=P) == -1 and "grad_residual" in err()
    assert call(b, okb, a9=None) == -1 and call(b, okb, a6=None) == -1
    assert L.cpab_b200_rms_norm_workspace(2, 100, 64) >= 64
    assert L.cpab_b200_rms_norm_workspace(9, 100, 64) == 0


def test_adamw_entry_point_validates():
    L = _native.lib()
    t = (_native._AdamWTensor * 1)()

    def one(**kw):
        base = dict(param=4096, grad=4096, exp_avg=4096, exp_avg_sq=4096, scales=None, step=4096,
                    lr_device=None, numel=8, dtype=0, state_bits=32, lr=1e-3, beta1=0.9, beta2=0.999,
                    eps=1e-8, weight_decay=0.0)
        for k, v in {**base, **kw}.items():
            setattr(t[0], k, v)
        return L.cpab_b200_adamw(ctypes.byref(t), 1, 0, P, None)

    assert one(dtype=5) == -1 and "dtype" in err()
    assert one(numel=-1) == -1 and "negative" in err()
    assert one(numel=(1 << 40) + 1) == -4
    assert one(step=None) == -1 and one(grad=None) == -1 and "null" in err()
    assert one(state_bits=16) == -1 and "bits" in err()
    assert one(state_bits=8) == -1 and "scales" in err()
    assert one(beta1=1.0) == -1 and "betas" in err()
    assert one(beta2=float("nan")) == -1
    assert one(eps=-1.0) == -1
    assert L.cpab_b200_adamw(None, 1, 0, P, None) == -1
    assert L.cpab_b200_adamw(ctypes.byref(t), 1, 0, None, None) == -1
    assert L.cpab_b200_adamw(ctypes.byref(t), -1, 0, P, None) == -1
    assert L.cpab_b200_adamw(None, 0, 0, P, None) == 0 and err() == ""


@pytest.fixture(params=["ext", "python"])
def path(request):
    if request.param == "python":
        with _ext.python_path():
            yield
    else:
        assert _ext.module() is not None
        yield


def test_cpu_tensors_are_refused(path):
    x, w = torch.randn(2, 3, 4), torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_scan_step(x[0], x[0], torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm(x, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        rms_norm_quantized(x, w)
    p, s = torch.zeros(4), torch.zeros(())
    with pytest.raises(RuntimeError, match="CUDA"):
        adamw_([p], [p], [p], [p], [s], lr=1e-3)


def test_whole_number_arguments_and_gradients_are_checked():
    x = torch.randn(2, 3, 4)
    with pytest.raises(TypeError, match="lengths"):
        gated_scan(x, x, lengths=torch.ones(2))
    with pytest.raises(TypeError, match="slots"):
        gated_scan_step(x[0], x[0], torch.zeros(3, 4), slots=torch.ones(3))
    with pytest.raises(RuntimeError, match="no gradient"):
        gated_scan_step(x[0].clone().requires_grad_(True), x[0], torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quantized(x, torch.ones(4, requires_grad=True))


def test_adamw_checks_its_options():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    q = torch.zeros(3)
    with pytest.raises(ValueError, match="lengths"):
        adamw_([q], [q, q], [q], [q], [q], lr=1e-3)
    with pytest.raises(ValueError, match="lr"):
        adamw_([q], [q], [q], [q], [q], lr=torch.tensor(1e-3))
    opt = AdamW(p)
    opt.step()                                         # no gradients: nothing to do
    assert p[0] not in opt.state or not opt.state[p[0]]


def test_a_norm_without_residual_has_its_inputs_type():
    L = _native.lib()
    a = [2, 0, 0, P, 8, None, 0, P, 4, 8, 1e-6, P, None, None, None]
    assert L.cpab_b200_rms_norm(*a) == -1 and "without a residual" in err()
    a = [2, 0, 0, P, 8, None, 0, P, 4, 8, 1e-6, P, P, None, None]
    assert L.cpab_b200_rms_norm_quantized(*a) == -1 and "without a residual" in err()


def test_a_learning_rate_on_another_device_is_refused(path):
    """By the call and by both of its native forms, before anything is launched
    (tensors without memory, so no GPU is needed)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        p, step, rate = (torch.empty(n, device=d) for n, d in ((4, "cuda:0"), (1, "cuda:0"), (1, "cuda:1")))
        with pytest.raises(ValueError, match="lr"):
            adamw_([p], [p], [p], [p], [step], lr=rate)
        ticket = torch.empty(1, device="cuda:0", dtype=torch.int32)
        fn = _native.adamw if _ext.module() is None else _ext.module().adamw
        with pytest.raises(RuntimeError, match="learning rate"):
            fn([p], [p], [p], [p], [], [step], [1], [0.0, 0.9, 0.999, 1e-8, 0.0], [rate], 0, ticket)


def test_a_group_on_two_devices_has_its_learning_rate_on_both(monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    from cpab import optim
    calls = []
    monkeypatch.setattr(optim, "_step", lambda groups, seed, workspace: calls.append((groups, workspace)))
    with FakeTensorMode():
        ps = [torch.nn.Parameter(torch.empty(5, device=d)) for d in ("cuda:0", "cuda:1", "cuda:0")]
        for p in ps:
            p.grad = torch.empty_like(p)
        rate = torch.empty((), device="cuda:0")
        AdamW(ps, lr=rate).step()
    assert len(calls) == 2
    for (group,), workspace in calls:
        params, lr = group[0], group[6]
        assert {t.device for t in (*params, lr, workspace)} == {params[0].device}
        assert (lr is rate) == (params[0].device == rate.device)


def test_the_seed_is_part_of_the_state_dict():
    p = torch.nn.Parameter(torch.zeros(3))
    opt = AdamW([p], state_bits=8, seed=7)
    two = AdamW([p], state_bits=8)
    assert two.seed == 0
    two.load_state_dict(opt.state_dict())
    assert two.seed == 7
    old = opt.state_dict()                                 # one without a seed leaves it alone
    del old["param_groups"][0]["seed"]
    three = AdamW([p], seed=9)
    three.load_state_dict(old)
    assert three.seed == 9
    three.seed = 2
    assert three.state_dict()["param_groups"][0]["seed"] == 2


def test_copies_and_pickles_of_adamw_step():
    """They come as far as the original: to the refusal of CPU tensors."""
    import copy
    import pickle
    p = torch.nn.Parameter(torch.zeros(3))
    opt = AdamW([p], lr=0.25, state_bits=8, seed=7)
    for twin in (opt, copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        (q,) = twin.param_groups[0]["params"]
        q.grad = torch.ones(3)
        assert twin.seed == 7 and twin.param_groups[0]["lr"] == 0.25
        with pytest.raises(RuntimeError, match="CUDA"):
            twin.step()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_state_dict_of_torchs_adamw(dtype):
    """Is taken: options that it lacks are the new optimizer's own, 16-bit moments
    become float32.  Options that this step does not have are refused."""
    p, q = (torch.nn.Parameter(torch.ones(6, 4, dtype=dtype)) for _ in range(2))
    theirs = torch.optim.AdamW([p, q], lr=3e-3, weight_decay=0.2)
    p.grad = torch.full_like(p, 0.5)                       # q has no gradient yet, so no state
    theirs.step()
    opt = AdamW([p, q], min_8bit_size=5, state_bits=8)
    opt.load_state_dict(theirs.state_dict())
    group = opt.param_groups[0]
    assert group["lr"] == 3e-3 and group["weight_decay"] == 0.2 and group["state_bits"] == 8
    state, want = opt.state[p], theirs.state[p]
    assert float(state["step"]) == 1
    for k in ("exp_avg", "exp_avg_sq"):
        assert state[k].dtype == torch.float32 and torch.equal(state[k], want[k].float())
    assert "scales" in opt._state(q, group)
    for option in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match=option):
            opt.load_state_dict(torch.optim.AdamW([p, q], **{option: True}).state_dict())
    assert opt.param_groups[0]["lr"] == 3e-3               # a refused one changes nothing
