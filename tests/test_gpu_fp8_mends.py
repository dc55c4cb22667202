"""Calls of the 8-bit operators at the ends of what they take: thresholds that broadcast."""
import pytest
import torch

from crosslayer_transcoder_b200 import fp8
from crosslayer_transcoder_b200.model import JumpReLU

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("layers, features", [(1, 1), (1, 40), (3, 1)])
@pytest.mark.parametrize("batch", [1, 50])
def test_thresholds_that_broadcast(layers, features, batch):
    """One threshold for all layers or features: the results and gradients of the eager definition."""
    torch.manual_seed(1)
    nl = JumpReLU(0.03, 0.7, layers, features).to(DEV)
    x = (torch.randn(batch, 3, 40, device=DEV) * 0.3).requires_grad_()
    g = torch.randint(-8, 9, x.shape, device=DEV).float()    # whole numbers: their sums are exact
    want, got = nl(x), nl(x, eight_bit=True)
    dx, dth = torch.autograd.grad(got, (x, nl.theta), g)
    wx = torch.autograd.grad(want, x, g)[0]
    assert torch.equal(got, want) and torch.equal(dx, wx) and dth.shape == nl.theta.shape
    th, bw = nl.theta.detach().double(), nl.bandwidth.double()
    inside = (x.double() > th - bw / 2) & (x.double() <= th + bw / 2)
    count = (g.double() * inside).sum_to_size(dth.shape)
    # the factor theta / bandwidth is rounded, then a product for each of the 120 thresholds at most, then their sum
    mags = (th / bw) * (g.double().abs() * inside).sum_to_size(dth.shape)
    assert bool(((dth.double() + (th / bw) * count).abs() <= 123 * 2.0 ** -24 * mags).all())
    fp8.check_status()
