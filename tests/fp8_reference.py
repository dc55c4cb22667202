"""The 8-bit format and operators in 64 bits, for the tests: plain torch on the CPU, no code of the package."""
import torch

EPS32 = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def scale_of(amax: float) -> float:
    """Smallest power of two s >= 2^-126 with amax / s <= 448; 1 for 0."""
    if amax == 0:
        return 1.0
    s = 2.0 ** -126
    while amax / s > 448:
        s *= 2
    return s


def quantize(x, rows):
    """(scales, values as they stand) of one matrix, block by block."""
    x = x.double().cpu()
    R, C = x.shape
    scales = torch.empty(-(-R // rows), -(-C // 128), dtype=torch.float64)
    out = torch.empty_like(x)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = (slice(i * rows, (i + 1) * rows), slice(j * 128, (j + 1) * 128))
            v = x[at]
            fin = v[torch.isfinite(v)].abs()
            s = scale_of(float(fin.max()) if fin.numel() else 0.0)
            scales[i, j] = s
            q = v / s
            e = torch.where(q == 0, torch.full_like(q, -6.0), torch.frexp(q)[1].double() - 1).clamp(min=-6)
            step = 2.0 ** (e - 3)
            r = torch.round(q / step) * step            # ties to even
            out[at] = torch.where(torch.isfinite(v), r, torch.full_like(r, float("nan"))) * s
    return scales, out


def rounded(x, rows=128):
    """x [Z, R, C] as its 8-bit form stands for it."""
    return torch.stack([quantize(m, rows)[1] for m in x]) if len(x) else x.double().cpu()


def sum_bound(K, mags):
    """How far an fp32 sum of K exactly representable products may be off the exact one: a step of 2^-23 (truncation) of the
    sum of magnitudes for each addition.  The tensor cores add 32 products at a time, at most 1024 to a sum (32 additions, with
    three more alignments each: 128); then come one addition a block and two scalings."""
    return (128 + -(-K // 128) + 2) * 2.0 ** -23 * mags


def check(got, want, mags, K, extra=0.0):
    """`got` is `want` (64 bits) within the bound of its sums and the rounding to its type."""
    g = got.detach().double().cpu()
    tol = sum_bound(K, mags) + HALF_STEP[got.dtype] * want.abs() * 1.01 + extra
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    bad = ~((g - want).abs() <= tol)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - want).abs() - tol)[bad].max()):.3g} over; "
                           f"first at {bad.nonzero()[0].tolist()}: {float(g[bad][0])} for {float(want[bad][0])}")
