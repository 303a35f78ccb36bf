"""orthogonalize, muon_ and Muon at the edges of what they take."""
import contextlib

import pytest
import torch

from cpab import _ext
from cpab.optim import Muon, muon_, orthogonalize
from test_gpu_muon import exact, matrices, most, off

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(params=["ext", "python"])
def path(request):
    with _ext.python_path() if request.param == "python" else contextlib.nullcontext():
        yield request.param


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sums_do_not_drift(dtype):
    """64 copies of a matrix side by side: their X X^T is the same as one's (64 and its
    root are powers of two), their result an eighth of one's, with the same roundings.  Only
    the sums are longer.  What an instruction cuts off them is a quarter of 2^-23 of the
    whole in the mean, which over the 512 of a segment comes to 1.5e-5 of A; the polynomial's
    slopes (1.2 of a change of A, 1.5 from step to step) make that 16 times as much."""
    g = torch.Generator(DEV).manual_seed(0)
    x = torch.randn(1700, 4096, device=DEV, generator=g).to(dtype)
    one = orthogonalize(x).double()
    many = orthogonalize(x.repeat(1, 64))[:, 4096 * 21:4096 * 22].double() * 8
    assert abs((one * many).sum() / (one * one).sum() - 1) <= 16 * 512 / 4 * 2.0 ** -23


@pytest.mark.parametrize("eps", [1e-3, 0.3, 1.0, 30.0, 1e6])
@pytest.mark.parametrize("shape", [(40, 70), (130, 260), (400, 300)])
def test_eps_near_and_above_the_norm(shape, eps, path):
    for dtype in (F32, BF16):
        x = matrices(shape, F32, 6)
        x = (x / x.norm()).to(dtype)
        assert off(orthogonalize(x, eps=eps), exact(x, eps=eps)) <= most(dtype, shape) + 2.0 ** -8 * (dtype == BF16)


@pytest.mark.parametrize("momentum", [0.95, 0.999, 0.99999, 1 - 2.0 ** -20])
@pytest.mark.parametrize("shape", [(20, 30), (130, 260), (131, 257)])
def test_momenta_keep_their_precision_near_1(shape, momentum, path):
    """1 - momentum is not the rounded momentum's: the new momentum is off by two
    products' and a sum's roundings and those of the two factors."""
    g, m = matrices(shape, F32, 1), matrices(shape, F32, 2) * 1e-3
    want = momentum * m.double() + (1 - momentum) * g.double()
    size = momentum * m.double().abs() + (1 - momentum) * g.double().abs()
    muon_([matrices(shape, F32, 3)], [g], [m], lr=0.1, momentum=momentum)
    assert ((m.double() - want).abs() <= 4 * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("shape", [(1, 7), (1, 70000), (300, 1)])
def test_values_on_their_way_from_far_below_eps_stay_in_range(shape, path):
    """A norm well under eps, and coefficients that let it grow by its cube's part alone
    and then move without rest, to 1.7 at most: 14 times the power of two that it began
    at, whose square is more than what is kept can be."""
    x = torch.zeros(shape, device=DEV)
    x.view(-1)[0] = 1.0
    for steps in (40, 56, 64):
        y = orthogonalize(x, steps, (1.0, 1.0, -0.5), 1 / 0.12 - 1)
        assert y.isfinite().all() and 0.1 < y.abs().max() <= 1.7


@pytest.mark.parametrize("shape", [(40, 70), (130, 260), (300, 280)])
def test_steps_from_far_below_eps(shape, path):
    """Steps that do not grow, or grow slowly, do not lose the bits of what is small."""
    x = matrices(shape, F32, 5)
    x = x / x.norm()
    for coefficients in ((1.0, 0.0, 0.0), (1.0, 1.0, -0.5), (1.5, -0.5, 0.0)):
        for eps in (4.0, 1e4, 1e9):
            for steps in (1, 6):
                y, want = orthogonalize(x, steps, coefficients, eps), exact(x, steps, coefficients, eps)
                assert off(y, want) <= 2 * most(F32, shape)


@pytest.mark.parametrize("dtype", [F32, torch.float64])
def test_a_learning_rate_on_the_cpu(dtype, path):
    """As torch's optimizer and its state dicts may have one; schedulers write into it."""
    a, b = (torch.nn.Parameter(matrices((20, 30), F32, 1)) for _ in range(2))
    lr = torch.tensor(0.25, dtype=dtype)
    ours, same = Muon([a], lr=lr), Muon([b], lr=0.25)
    for rate in (0.25, 0.5):
        lr.fill_(rate)
        same.param_groups[0]["lr"] = rate
        a.grad = matrices((20, 30), F32, 2)
        b.grad = a.grad.clone()
        ours.step()
        same.step()
        assert torch.equal(a, b)
    theirs = torch.optim.Muon([torch.nn.Parameter(a.detach().clone())], lr=torch.tensor(0.5))
    theirs.param_groups[0]["params"][0].grad = a.grad.clone()
    theirs.step()
    ours.load_state_dict(theirs.state_dict())
    ours.step()
    with pytest.raises(ValueError, match="one element"):
        Muon([a], lr=torch.zeros(2))


def in_a_bucket(tensors, lead):
    """The tensors as views into one flat buffer, `lead` elements from its beginning."""
    flat = torch.zeros(lead + sum(t.numel() + 1 for t in tensors), device=DEV, dtype=tensors[0].dtype)
    views, at = [], lead
    for t in tensors:
        views.append(flat[at:at + t.numel()].view(t.shape).copy_(t))
        at += t.numel() + 1
    return views


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lead", [0, 1, 3])
def test_views_into_a_flat_bucket(lead, dtype, path):
    """Parameters, gradients and momenta off 16 bytes whose rows are whole vectors, as
    data-parallel training makes them: the same step as of tensors of their own."""
    shapes = [(130, 264), (264, 130), (304, 296), (296, 304), (16, 24), (136, 8), (1, 40)]
    ps, gs = ([matrices(s, dtype, k + at, 0.05) for k, s in enumerate(shapes)] for at in (0, 20))
    ms = [matrices(s, F32, k + 40) for k, s in enumerate(shapes)]
    views = [in_a_bucket(ts, lead) for ts in (ps, gs, ms)]
    for lists in ((ps, gs, ms), views):
        for _ in range(2):
            muon_(*lists, lr=0.1, momentum=0.9)
    for own, seen in zip((ps, gs, ms), views):
        assert all(torch.equal(a, b) for a, b in zip(own, seen))
    for x in ps:
        (view,) = in_a_bucket([x], lead + 1)
        assert torch.equal(orthogonalize(view), orthogonalize(x))
