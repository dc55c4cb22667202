"""Calls of the 8-bit operators at the ends of what they take: thresholds that broadcast, scales that are no powers of two,
scales whose products fp32 does not hold."""
import numpy as np
import pytest
import torch

from crosslayer_transcoder_b200 import fp8
from crosslayer_transcoder_b200.model import JumpReLU
from tests import fp8_reference as ref

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


# ---- products of scales outside of fp32's normal numbers -----------------------------------------------------------------------
def _scales(shape, low, high, g):
    """Numbers of any mantissa with exponents from `low` to `high`."""
    return ((1 + torch.rand(shape, generator=g).double()) * 2.0 ** torch.randint(low, high + 1, shape, generator=g)).float()


def _far_operands(kind, M, K, N, rows, a_t, b_t, g):
    kb = -(-K // 128)
    va, vb = torch.randn(M, K, generator=g), torch.randn(K, N, generator=g)
    sa, sb = (-(-M // rows), kb), (kb, -(-N // 128))
    if kind == "small":                                         # products of 2^-156 to 2^-134
        va, vb = va * 100, vb * 100
        sa, sb = _scales(sa, -106, -94, g), _scales(sb, -50, -40, g)
    else:                                                       # of 2^128 to 2^134, and values of 2^-9 or 0
        va, vb = va.sign() * (va.abs() > 1) * 2.0 ** -9, vb.sign() * (vb.abs() > 1) * 2.0 ** -9
        sa, sb = _scales(sa, 60, 62, g), _scales(sb, 68, 70, g)
    zero = slice(M // 2, M // 2 + (M > 1))
    va[zero] = 0                                                # a row of zeros
    va, vb = va.clamp(-448, 448).to(torch.float8_e4m3fn), vb.clamp(-448, 448).to(torch.float8_e4m3fn)
    da = va.double() * sa.double().repeat_interleave(rows, 0)[:M].repeat_interleave(128, 1)[:, :K]
    db = vb.double() * sb.double().repeat_interleave(128, 0)[:K].repeat_interleave(128, 1)[:, :N]
    t = lambda v, s, r, turned: (fp8.BlockTensor(v.t().contiguous().to(DEV), s.t().contiguous().to(DEV), r).mT if turned else
                                 fp8.BlockTensor(v.to(DEV), s.to(DEV), r))
    return t(va, sa, rows, a_t), t(vb, sb, 128, b_t), da, db, zero


@pytest.mark.parametrize("layout", [(1, False, False), (128, False, False), (1, False, True), (128, True, False), (128, True, True)])
@pytest.mark.parametrize("shape", [(70, 300, 140), (1, 5000, 72), (2500, 640, 2600), (257, 1024, 33)])
@pytest.mark.parametrize("kind", ["small", "large"])
def test_scales_whose_product_fp32_does_not_hold(kind, shape, layout):
    M, K, N = shape
    a, b, da, db, zero = _far_operands(kind, M, K, N, *layout, torch.Generator().manual_seed(11))
    want, mags = da @ db, da.abs() @ db.abs()
    assert float(mags.max()) < 2.0 ** 127 and float(mags.max()) > 2.0 ** -126      # results are numbers of fp32
    for out in (torch.float32, torch.bfloat16):
        y = fp8.matmul(a, b, out_dtype=out)
        # below 2^-126 each addition (one a block, and one a part) and the last rounding are off by half of the least number
        least = 2.0 ** -149 if out == torch.float32 else 2.0 ** -133
        ref.check(y, want, mags, K, extra=(-(-K // 128) * 2 + 2) * 2.0 ** -150 + least / 2)
        assert not y[zero].any()
    fp8.check_status()


def test_rows_of_small_ordinary_and_large_scales():
    """Side by side in a warp; zero, infinite and NaN scales reach their own rows alone."""
    M, K, N = 96, 384, 260
    g = torch.Generator().manual_seed(12)
    va = (torch.randn(M, K, generator=g).sign() * 2.0 ** -9).to(torch.float8_e4m3fn)
    vb = (torch.randn(K, N, generator=g).sign() * 2.0 ** -9).to(torch.float8_e4m3fn)
    sb = torch.full((3, 3), 1.5 * 2.0 ** 20)
    sa = torch.tensor([2.0 ** -149, 1.1 * 2.0 ** -147, 1.7 * 2.0 ** 115, 1.0, 0.0, 2.0 ** 108, 3.0, 1.3 * 2.0 ** -146])[:, None].repeat(12, 3)
    sa[17, 1], sa[40, 2] = float("inf"), float("nan")
    y = fp8.matmul(fp8.BlockTensor(va.to(DEV), sa.to(DEV), 1), fp8.BlockTensor(vb.to(DEV), sb.to(DEV)), out_dtype=torch.float32).cpu()
    bad = torch.zeros(M, dtype=torch.bool)
    bad[17] = bad[40] = True
    da, db = va.double() * sa.double().repeat_interleave(128, 1), vb.double() * sb.double().repeat_interleave(128, 0)[:, :1]
    ref.check(y[~bad], da[~bad] @ db, da[~bad].abs() @ db.abs(), K, extra=10 * 2.0 ** -149)
    assert not y[4::8].any() and not y[bad].isfinite().any()


@pytest.mark.parametrize("large", [False, True])
def test_passes_of_small_and_large_numbers(large):
    """Blocks whose scales have a product of 2^-152, or of 2^129 (from one row and one column), and results that are numbers of fp32."""
    B, D, F = 40, 2001, 72
    g = torch.Generator().manual_seed(13)
    x, W = torch.rand(B, 1, D, generator=g) * 0.5 + 0.5, torch.rand(1, D, F, generator=g) * 0.5 + 0.5
    x, W = (x * 2.0 ** 112, W * 2.0 ** 3) if large else (x * 2.0 ** -80, W * 2.0 ** -56)
    x[0] = 0
    if large:
        x[1], W[:, :, 0] = 2.0 ** 127, 2.0 ** 18
    y = fp8.project(x.to(DEV), W.to(DEV)).cpu()
    xq, wq = ref.rounded(x.transpose(0, 1)), ref.rounded(W)
    want = (xq @ wq).transpose(0, 1)
    fits = want < 2.0 ** 127.9
    assert float(fits.double().mean()) > 0.9 and float(want[fits].max()) > 2.0 ** -126
    at = lambda t: torch.where(fits, t, torch.zeros_like(t))
    ref.check(at(y), at(want), at(want), D, extra=40 * 2.0 ** -150)
    assert not y[0].any()
