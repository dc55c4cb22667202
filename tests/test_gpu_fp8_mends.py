"""Calls of the 8-bit operators at the ends of what they take: thresholds that broadcast, scales that are no powers of two."""
import numpy as np
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


# ---- read-back at any scale --------------------------------------------------------------------------------------------------
CODES = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.float8_e4m3fn)


def once(x, dtype):
    """float64 to `dtype`, rounded once to nearest, ties to even (torch's own conversion of fp64 to 16 bits goes through fp32)."""
    if dtype != torch.bfloat16:
        with np.errstate(over="ignore"):
            return torch.from_numpy(x.numpy().astype(np.float16 if dtype == torch.float16 else np.float32))
    step = 2.0 ** (torch.frexp(x)[1].clamp(min=-125).double() - 8)      # of 8 bits; below 2^-126 the least number, 2^-133
    r = torch.where(x.isfinite(), torch.round(x / step) * step, x)
    return r.float().to(torch.bfloat16)                                 # exact, or too large for both


def _near_borders(dtype):
    """Scales whose product with some code is next to the middle of two neighbours of `dtype`: rounding to fp32 first moves many of
    them onto it.  Subnormal and large ones, and ordinary numbers, too."""
    g = torch.Generator().manual_seed(7)
    n, bits = 3000, 11 if dtype == torch.float16 else 8
    code = CODES[:127].double()[torch.randint(1, 127, (n,), generator=g)]
    middle = (torch.randint(2 ** (bits - 1), 2 ** bits, (n,), generator=g).double() + 0.5) * 2.0 ** torch.randint(-30, 2, (n,), generator=g)
    odd = torch.tensor([2.0 ** -149, 3 * 2.0 ** -149, 12345 * 2.0 ** -149, 1.3 * 2.0 ** -126, 2.0 ** -126, 3.4e38, 2.0 ** 127, 0.0, 1.0, 0.1,
                        -0.3, float("inf"), float("nan"), 1.7 * 2.0 ** -133, 1.9 * 2.0 ** -24, 1e-7, 1e-8, 150.0, 1.1e35])
    near = (middle / code).float()
    tiny = (2.0 ** -133 * (torch.randint(1, 64, (200,), generator=g).double() + 0.5) / CODES[:127].double()[torch.randint(1, 127, (200,), generator=g)]).float()
    return torch.cat([near, near * (1 + 2.0 ** -23), tiny, odd])


def test_near_borders_are_such():
    """Without the wider product many of the inputs below are wrong: the test sees the difference."""
    for dtype in (torch.float16, torch.bfloat16):
        s = _near_borders(dtype)
        exact = CODES.double()[None] * s.double()[:, None]
        twice = (CODES.float()[None] * s[:, None]).to(dtype)
        assert int((twice != once(exact, dtype)).logical_and(~exact.isnan()).sum()) > 500


@pytest.mark.parametrize("columns", [256, 255, 129, 16, 7])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_read_back_is_rounded_once(dtype, columns):
    """Every code, at aligned rows and others, with any scales."""
    s = _near_borders(dtype)
    for start in range(0, 256, columns):
        codes = CODES[start:start + columns] if start + columns <= 256 else CODES[256 - columns:]
        scales = s[:, None].expand(-1, -(-columns // 128)).clone()
        scales[:, -1] = scales[:, -1].roll(1)                # (two scales in a row, where there are two blocks)
        q = fp8.BlockTensor(codes.expand(len(s), columns).contiguous().to(DEV), scales.to(DEV), block_rows=1)
        got = q.dequantize(dtype).cpu()
        want = once(codes.double()[None] * scales.double().repeat_interleave(128, 1)[:, :columns], dtype)
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
