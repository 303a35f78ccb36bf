"""SeriesLocalizer: a stream's answers are those of the whole series, with 8-bit
projections too."""
import pytest
import torch

from cpab.pytorch.localizer import SeriesLocalizer

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]
DEV = "cuda"


@pytest.mark.parametrize("width", [33, 64, 200])
@pytest.mark.parametrize("bits", [16, 8])
def test_a_stream_answers_with_the_projections_of_the_network(bits, width):
    """Both are given by the same codes, but where a value that differs by float32's
    roundings (2^-20 after some tens of operations) lies that near to a border between
    codes, a share of 2^-20 / 2^-4 of them, and is then off by a code's 2^-4:
    2^-4 sqrt(2^-16) = 2^-12 of a projection; four of them and twice that."""
    torch.manual_seed(0)
    net = SeriesLocalizer(3, 11, width, 2, projection_bits=bits).to(DEV)
    torch.nn.init.normal_(net.head.weight, std=0.3)
    x = torch.randn(4, 3, 60, generator=torch.Generator().manual_seed(1)).to(DEV)
    states = net.new_states(4)
    for t in range(60):
        theta = net.step(x[:, :, t], states)
    with torch.no_grad():
        whole = net(x)
    assert (theta - whole).norm() <= 8 * 2.0 ** -12 * whole.norm()
