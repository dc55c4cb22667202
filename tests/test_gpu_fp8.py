"""8-bit operands and checkpoints against their definitions in 64 bits (tests/fp8_reference.py)."""
import pytest
import torch

from crosslayer_transcoder_b200 import fp8
from tests import fp8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _rand(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x *= torch.exp(torch.randn(shape[-1], generator=g))       # columns of different spread
    return (x * scale).to(dtype).to(DEV)


# ---- quantisation ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 768), (2, 128, 128), (3, 129, 257), (1, 300, 15), (2, 5, 1000), (1, 4001, 72)])
def test_quantize(shape, rows, dtype):
    x = _rand(shape, 1, dtype=dtype)
    q = fp8.quantize(x, block_rows=rows)
    assert q.shape == x.shape and q.values.dtype == torch.float8_e4m3fn
    for z in range(shape[0]):
        s, v = ref.quantize(x[z], rows)
        assert torch.equal(q.scales[z].double().cpu(), s)
        assert torch.equal((q.values[z].float().cpu().double() * s.repeat_interleave(rows, 0)[:shape[1]].repeat_interleave(128, 1)[:, :shape[2]]), v)
    for out in TYPES:
        back = q.dequantize(out)
        want = torch.stack([ref.quantize(m, rows)[1] for m in x]).to(out)
        assert torch.equal(back.cpu(), want)
    fp8.check_status()


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_borders(rows):
    """Amaxes at and beside the scale's borders, zeros, subnormals, the largest numbers, ties between e4m3 neighbours."""
    x = torch.zeros(128 * 3, 128 * 4)
    for j, top in enumerate([448.0, 448.0 * (1 + 2 ** -20), 2.0 ** -149, 3.4e38]):
        x[0, 128 * j] = top
        x[1, 128 * j + 1] = -top
    ties = torch.tensor([1.0625, 1.1875, -1.0625, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 448.0, 432.0, 464.0 - 2 ** -10])
    x[130, :10] = ties
    x[140, 130:140] = ties * 2.0 ** -30
    x[300, 256:] = torch.arange(256) * 2.0 ** -12
    x = x.to(DEV)
    s, v = ref.quantize(x, rows)
    q = fp8.quantize(x, block_rows=rows)
    assert torch.equal(q.scales.double().cpu(), s)
    # rounded to fp32: 3.4e38 became 256 * 2^120 = 2^128, which fp32 does not hold
    assert torch.equal(q.dequantize().cpu(), v.float())


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_not_finite(rows, dtype):
    x = _rand((1, 140, 200), 3, dtype=dtype)
    x[0, 3, 5], x[0, 4, 6], x[0, 130, 150] = float("inf"), float("-inf"), float("nan")
    x[0, 7, 128:] = float("nan")                     # a block without a finite value
    s, v = ref.quantize(x[0], rows)
    q = fp8.quantize(x, block_rows=rows)
    assert torch.equal(q.scales[0].double().cpu(), s)
    assert torch.equal(torch.nan_to_num(q.dequantize()[0].double().cpu(), nan=-7.0), torch.nan_to_num(v, nan=-7.0))


def test_quantize_strides():
    """Views: rows at a distance, layers inside, misaligned starts, broadcasts, transposed (copied)."""
    base = _rand((40, 3, 200), 4)
    for x in (base.transpose(0, 1), base[:, 1, 3:150], base[1:, :, 1:], base[:, :1].expand(40, 5, 200), base[0, 0].expand(3, 130, 200),
              base[:, 0].t(), base[:, :, :1], base.half()[:, 2, 1:100]):
        a, b = fp8.quantize(x), fp8.quantize(x.contiguous())
        assert torch.equal(a.scales, b.scales) and torch.equal(a.values.float(), b.values.float())
    assert fp8.quantize(base[:0]).dequantize().shape == (0, 3, 200)
    assert fp8.quantize(base[0, :, :0]).dequantize().shape == (3, 0)


def test_copy_of_a_copy():
    x = _rand((2, 200, 300), 5)
    for rows in (1, 128):
        back = fp8.quantize(x, rows).dequantize()
        assert torch.equal(fp8.quantize(back, rows).dequantize(), back)


# ---- product -----------------------------------------------------------------------------------------------------------------
def _operands(G, M, K, N, rows, a_t, b_t, seed):
    xa = _rand((G, K, M) if a_t else (G, M, K), seed)
    xb = _rand((G, N, K) if b_t else (G, K, N), seed + 1)
    a, b = fp8.quantize(xa, rows), fp8.quantize(xb)
    va, vb = ref.rounded(xa, rows), ref.rounded(xb)
    return (a.mT if a_t else a, b.mT if b_t else b, va.transpose(1, 2) if a_t else va, vb.transpose(1, 2) if b_t else vb)


SHAPES = [(1, 1, 1, 1), (1, 1, 128, 256), (1, 128, 128, 256), (1, 7, 300, 33), (2, 129, 255, 257), (3, 200, 640, 130), (1, 300, 17, 520),
          (1, 1, 5000, 72), (2, 260, 2048, 96)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("layout", [(1, False, False), (128, False, False), (1, False, True), (128, True, False), (128, True, True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_matmul(shape, layout, out):
    G, M, K, N = shape
    a, b, va, vb = _operands(G, M, K, N, *layout, seed=10)
    bias = _rand((G, N), 12) if K % 2 else None
    y = fp8.matmul(a, b, bias=bias, out_dtype=out)
    assert y.shape == (G, M, N) and y.dtype == out
    want = va @ vb + (0 if bias is None else bias.double().cpu()[:, None])
    mags = va.abs() @ vb.abs() + (0 if bias is None else bias.abs().double().cpu()[:, None])
    ref.check(y, want, mags, K)
    fp8.check_status()


@pytest.mark.parametrize("shape", [(12, 700, 768, 1500), (1, 4000, 768, 2600), (4, 1030, 300, 1024)])
@pytest.mark.parametrize("layout", [(1, False, False), (128, True, False), (128, False, True), (128, True, True)])
def test_matmul_pairs(shape, layout):
    """Sizes at which clusters of two CTAs run, with ragged rows and columns."""
    G, M, K, N = shape
    g = torch.Generator(device=DEV).manual_seed(3)
    rows, a_t, b_t = layout
    xa = torch.randn((G, K, M) if a_t else (G, M, K), generator=g, device=DEV)
    xb = torch.randn((G, N, K) if b_t else (G, K, N), generator=g, device=DEV)
    a, b = fp8.quantize(xa, rows), fp8.quantize(xb)
    va, vb = a.dequantize().double(), b.dequantize().double()         # (tested above)
    va, vb = (va.mT if a_t else va), (vb.mT if b_t else vb)
    y = fp8.matmul(a.mT if a_t else a, b.mT if b_t else b, out_dtype=torch.float32)
    tol = ref.sum_bound(K, va.abs() @ vb.abs()) + ref.EPS32 * (va @ vb).abs()
    assert bool(((y.double() - va @ vb).abs() <= tol).all())
    fp8.check_status()


def test_matmul_any_scales_and_strides():
    """Scales that are no powers of two, values from another tensor's middle, rows that are not 16-byte aligned (copied)."""
    g = torch.Generator().manual_seed(0)
    M, K, N = 70, 333, 140
    va = torch.randn(M, K + 5, generator=g).to(torch.float8_e4m3fn)
    vb = torch.randn(K, N + 3, generator=g).to(torch.float8_e4m3fn)
    sa, sb = torch.rand(M, 3, generator=g) + 0.1, torch.rand(3, 2, generator=g) + 0.1
    a = fp8.BlockTensor(va.to(DEV)[:, 2:K + 2], sa.to(DEV), block_rows=1)
    b = fp8.BlockTensor(vb.to(DEV)[:, 1:N + 1], sb.to(DEV).t().contiguous().t())
    y = fp8.matmul(a, b, out_dtype=torch.float32)
    da = va[:, 2:K + 2].double() * sa.double().repeat_interleave(128, 1)[:, :K]
    db = vb[:, 1:N + 1].double() * sb.double().repeat_interleave(128, 0)[:K].repeat_interleave(128, 1)[:, :N]
    ref.check(y, da @ db, da.abs() @ db.abs(), K)
    assert torch.equal(a.dequantize().cpu(), (va[:, 2:K + 2].float() * sa.repeat_interleave(128, 1)[:, :K]))


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 17), (2, 3, 15), (3, 5, 129), (1, 40, 333), (2, 129, 1001)])
@pytest.mark.parametrize("start", [0, 1, 2, 3, 7])
def test_matmul_rows_that_start_anywhere(shape, start):
    """Values without a gap between rows, from any address, broadcast over the stack or not, as either operand."""
    Z, R, C = shape
    g = torch.Generator().manual_seed(1)
    flat = torch.randn(Z * R * C + 16, generator=g).to(torch.float8_e4m3fn).to(DEV)
    v = flat[start:start + Z * R * C].view(Z, R, C)
    s = torch.ones(Z, 1 + (R - 1) // 128, 1 + (C - 1) // 128, device=DEV)
    for values in (v, v[:1].expand(Z, R, C), v.mT):
        sc = s if values.shape == v.shape else torch.ones(Z, 1 + (C - 1) // 128, 1 + (R - 1) // 128, device=DEV)
        b = fp8.BlockTensor(values, sc)
        dense = values.float()
        other = fp8.quantize(torch.randint(-4, 5, (Z, 24, values.shape[1]), generator=g).float().to(DEV))
        y = fp8.matmul(other, b, out_dtype=torch.float32)
        ref.check(y, (other.dequantize() .double() @ dense.double()).cpu(), (other.dequantize().double().abs() @ dense.double().abs()).cpu(), R)
        y = fp8.matmul(b, fp8.quantize(torch.ones(Z, values.shape[2], 3, device=DEV)), out_dtype=torch.float32)
        ref.check(y, dense.double().cpu().sum(2, keepdim=True).expand(-1, -1, 3), dense.double().cpu().abs().sum(2, keepdim=True).expand(-1, -1, 3), C)


def test_matmul_not_finite():
    """NaN reaches its row or column and nothing else; infinite and NaN elements behind the matrix's end are not read."""
    a, b = _rand((1, 130, 200), 1), _rand((1, 200, 140), 2)
    clean = fp8.matmul(fp8.quantize(a, 1), fp8.quantize(b), out_dtype=torch.float32)
    a[0, 129, 199] = float("nan")
    y = fp8.matmul(fp8.quantize(a, 1), fp8.quantize(b), out_dtype=torch.float32)
    assert torch.isnan(y[0, 129]).all() and torch.equal(y[0, :129], clean[0, :129])


@pytest.mark.parametrize("zero", [0, 1, 2, 3])
def test_matmul_empty(zero):
    dims = [2, 3, 4, 5]
    dims[zero] = 0
    G, M, K, N = dims
    a, b = fp8.quantize(torch.zeros(G, M, K, device=DEV), 1), fp8.quantize(torch.zeros(G, K, N, device=DEV))
    bias = torch.randn(N, device=DEV)
    y = fp8.matmul(a, b, bias, out_dtype=torch.float32)
    assert y.shape == (G, M, N) and torch.equal(y, bias.expand(G, M, N))


def test_matmul_repeats_and_matrices():
    """Few rows over a long axis (cut into parts) give the same bits every time; matrices and stacks of one agree."""
    a, b, va, vb = _operands(1, 33, 20000, 200, 1, False, False, seed=3)
    first = fp8.matmul(a, b, out_dtype=torch.float32)
    for _ in range(3):
        assert torch.equal(fp8.matmul(a, b, out_dtype=torch.float32), first)
    assert torch.equal(fp8.matmul(a[0], b[0], out_dtype=torch.float32), first[0])
    ref.check(first, va @ vb, va.abs() @ vb.abs(), 20000)


# ---- projection --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(1, 1, 1, 1), (1, 2, 64, 256), (136, 3, 64, 256), (200, 2, 129, 77), (130, 1, 320, 2001)])
def test_project(dims, dtype):
    B, L, D, F = dims
    x = _rand((B, L, D), 1, dtype=dtype).requires_grad_()
    W = _rand((L, D, F), 2, D ** -0.5).requires_grad_()
    b = _rand((L, F), 3).requires_grad_()
    g = _rand((B, L, F), 4, 1e-2, dtype)
    y = fp8.project(x, W, b)
    dx, dW, db = torch.autograd.grad(y, (x, W, b), g)
    assert (y.dtype, dx.dtype, dW.dtype, db.dtype) == (dtype, dtype, torch.float32, torch.float32)
    xq, wq, gq = (ref.rounded(t.detach().transpose(0, 1)) for t in (x, W.transpose(0, 1), g))
    bias = b.detach().double().cpu()
    ref.check(y.transpose(0, 1), xq @ wq + bias[:, None], xq.abs() @ wq.abs() + bias.abs()[:, None], D)
    ref.check(dx.transpose(0, 1), gq @ wq.mT, gq.abs() @ wq.abs().mT, F)
    ref.check(dW, xq.mT @ gq, xq.abs().mT @ gq.abs(), B)
    gd = g.double().cpu()
    assert bool(((db.double().cpu() - gd.sum(0)).abs() <= (B + 2) * 2.0 ** -24 * gd.abs().sum(0)).all())
    fp8.check_status()


def test_project_forms():
    """One layer, leading axes, no bias, gradients of some operands only, 16-bit weights, an expanded gradient, no rows."""
    x, W, b = _rand((4, 5, 96), 1), _rand((96, 130), 2, 0.1), _rand((130,), 3)
    y = fp8.project(x, W, b)
    assert torch.equal(y, fp8.project(x.view(20, 1, 96), W[None], b[None]).view(4, 5, 130))
    assert torch.equal(fp8.project(x, W), fp8.project(x, W, torch.zeros_like(b)))
    assert not y.requires_grad
    full = [t.clone().requires_grad_() for t in (x, W, b)]
    grads = torch.autograd.grad(fp8.project(*full).sum(), full)         # an expanded gradient
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, W, b))]
        assert torch.equal(torch.autograd.grad(fp8.project(*some).sum(), some[i])[0], grads[i])
    Wh = W.bfloat16().requires_grad_()
    dW = torch.autograd.grad(fp8.project(x, Wh, b).sum(), Wh)[0]
    assert dW.dtype == torch.bfloat16
    empty = x[:0].clone().requires_grad_()
    Wr = W.clone().requires_grad_()
    br = b.clone().requires_grad_()
    out = fp8.project(empty, Wr, br)
    de, dW, db = torch.autograd.grad(out, (empty, Wr, br), torch.zeros_like(out))
    assert out.shape == (0, 5, 130) and de.shape == empty.shape and not dW.any() and not db.any()


def test_project_broadcast_input():
    """An input that is broadcast gets the sum of its copies' gradients."""
    row = _rand((1, 2, 64), 1).requires_grad_()
    W = _rand((2, 64, 40), 2, 0.1)
    y = fp8.project(row.expand(9, 2, 64), W)
    g = torch.ones_like(y)
    full = row.detach().expand(9, 2, 64).clone().requires_grad_()
    want = torch.autograd.grad(fp8.project(full, W), full, g)[0].sum(0, keepdim=True)
    assert torch.allclose(torch.autograd.grad(y, row, g)[0], want, rtol=1e-6, atol=0)


def _small_integers(shape, seed, top=7):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).float().to(DEV)


def test_gradients_against_differences():
    """Operands that e4m3 holds exactly: the passes are then linear in each of them, and a difference of outputs is the gradient."""
    B, L, D, F = 5, 2, 20, 30
    x, W, b, g = _small_integers((B, L, D), 1), _small_integers((L, D, F), 2), _small_integers((L, F), 3), _small_integers((B, L, F), 4)
    leaves = [t.clone().requires_grad_() for t in (x, W, b)]
    grads = torch.autograd.grad(fp8.project(*leaves), leaves, g)
    for i, at in ((0, (3, 1, 7)), (0, (4, 0, 19)), (1, (1, 0, 29)), (1, (0, 19, 0)), (2, (1, 2))):
        lo, hi = [t.clone() for t in (x, W, b)], [t.clone() for t in (x, W, b)]
        lo[i][at] -= 1
        hi[i][at] += 1
        diff = ((fp8.project(*hi) - fp8.project(*lo)) * g).sum() / 2
        assert float(diff) == float(grads[i][at])
    f, ws, bd, gd = _small_integers((B, 3, F), 5), [_small_integers((t + 1, F, D), 6 + t) for t in range(3)], _small_integers((3, D), 9), _small_integers((B, 3, D), 10)
    leaves = [t.clone().requires_grad_() for t in (f, bd, *ws)]
    grads = torch.autograd.grad(fp8.crosslayer_decode(leaves[0], leaves[2:], leaves[1]), leaves, gd)
    for i, at in ((0, (0, 0, 3)), (0, (4, 2, 29)), (1, (2, 5)), (2, (0, 1, 1)), (4, (1, 29, 19)), (4, (2, 0, 0))):
        lo, hi = [t.clone() for t in (f, bd, *ws)], [t.clone() for t in (f, bd, *ws)]
        lo[i][at] -= 1
        hi[i][at] += 1
        diff = ((fp8.crosslayer_decode(hi[0], hi[2:], hi[1]) - fp8.crosslayer_decode(lo[0], lo[2:], lo[1])) * gd).sum() / 2
        assert float(diff) == float(grads[i][at])


# ---- crosslayer decoder --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dims", [(1, 1, 1, 1), (1, 2, 40, 64), (136, 3, 256, 64), (131, 4, 201, 77), (260, 2, 640, 320)])
def test_crosslayer_decode(dims, dtype):
    B, L, F, D = dims
    f = torch.relu(_rand((B, L, F), 1)).to(dtype).requires_grad_()
    ws = [_rand((t + 1, F, D), 2 + t, 0.1).requires_grad_() for t in range(L)]
    b = _rand((L, D), 30).requires_grad_()
    g = _rand((B, L, D), 31, 1e-2, dtype)
    y = fp8.crosslayer_decode(f, ws, b)
    df, db, *dW = torch.autograd.grad(y, (f, b, *ws), g)
    fq, gq, wq = ref.rounded(f.detach().transpose(0, 1)), ref.rounded(g.transpose(0, 1)), [ref.rounded(w.detach()) for w in ws]
    for t in range(L):
        bias = b[t].detach().double().cpu()
        ref.check(y[:, t], (fq[:t + 1] @ wq[t]).sum(0) + bias, (fq[:t + 1].abs() @ wq[t].abs()).sum(0) + bias.abs(), (t + 1) * F)
        ref.check(dW[t], fq[:t + 1].mT @ gq[t], fq[:t + 1].abs().mT @ gq[t].abs(), B)
        ref.check(df[:, t], sum(gq[u] @ wq[u][t].mT for u in range(t, L)), sum(gq[u].abs() @ wq[u][t].abs().mT for u in range(t, L)),
                  (L - t) * D)
    gd = g.double().cpu()
    assert bool(((db.double().cpu() - gd.sum(0)).abs() <= (B + 2) * 2.0 ** -24 * gd.abs().sum(0)).all())
    fp8.check_status()


def test_crosslayer_decode_block_forms():
    """Blocks that are views, of mixed types or many give what contiguous fp32 ones do."""
    L, F, D, B = 3, 72, 40, 30
    f, b = torch.relu(_rand((B, L, F), 1)), _rand((L, D), 2)
    wide = [_rand((t + 1, F, 2 * D), 3 + t).bfloat16().float() for t in range(L)]
    views = [w[:, :, ::2] for w in wide]
    want = fp8.crosslayer_decode(f, [v.contiguous() for v in views], b)
    assert torch.equal(fp8.crosslayer_decode(f, views, b), want)
    mixed = [v.contiguous().to(torch.bfloat16 if t == 1 else torch.float32).requires_grad_() for t, v in enumerate(views)]
    y = fp8.crosslayer_decode(f, mixed, b)
    assert torch.equal(y, want)
    grads = torch.autograd.grad(y, mixed, torch.ones_like(y))
    assert [g.dtype for g in grads] == [torch.float32, torch.bfloat16, torch.float32]
    assert torch.equal(fp8.crosslayer_decode(f.view(5, 6, L, F), views, b), want.view(5, 6, L, D))
    L = 66
    f, ws = torch.relu(_rand((4, L, 8), 1)), [_rand((t + 1, 8, 16), t) for t in range(L)]
    y = fp8.crosslayer_decode(f, ws)
    fq, wq = ref.rounded(f.transpose(0, 1)), ref.rounded(ws[-1])
    ref.check(y[:, -1], (fq @ wq).sum(0), (fq.abs() @ wq.abs()).sum(0), L * 8)
    fp8.check_status()


@pytest.mark.parametrize("needs", ["f", "b", "blocks", "one block", "f and b"])
def test_crosslayer_decode_gradients_of_some(needs):
    """What needs no gradient gets none, and the others' are the same bits as when all are asked for."""
    L, F, D = 3, 40, 24
    f, b = _rand((50, L, F), 1), _rand((L, D), 2)
    blocks = [_rand((t + 1, F, D), 3 + t) for t in range(L)]
    g = _rand((50, L, D), 9)
    every = [x.clone().requires_grad_() for x in (f, b, *blocks)]
    want = torch.autograd.grad(fp8.crosslayer_decode(every[0], every[2:], every[1]), every, g)
    at = {"f": [0], "b": [1], "blocks": [2, 3, 4], "one block": [3], "f and b": [0, 1]}[needs]
    some = [x.clone().requires_grad_(i in at) for i, x in enumerate((f, b, *blocks))]
    fp8.crosslayer_decode(some[0], some[2:], some[1]).backward(g)
    for i, x in enumerate(some):
        assert torch.equal(x.grad, want[i]) if i in at else x.grad is None


# ---- (Jump)ReLU ----------------------------------------------------------------------------------------------------------------
def _jump_reference(x, theta, bw, g):
    x, g, th = x.double().cpu(), g.double().cpu(), theta.double().cpu()
    y = torch.where((x > th) & (x > 0), x, torch.zeros_like(x))
    y = torch.where(torch.isnan(x), x, y)
    inside = (x > th - bw / 2) & (x <= th + bw / 2)
    s = torch.where(inside, g, torch.zeros_like(g))
    dims = tuple(range(x.dim() - th.dim()))
    return y, torch.where(x < 0, torch.zeros_like(g), g), -(th / bw) * s.sum(dims), (th / bw).abs() * s.abs().sum(dims)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 3, 8), (200, 3, 256), (777, 2, 201), (33, 1, 4103), (5000, 16)])
def test_jump_relu(shape, dtype):
    x = _rand(shape, 1, 0.5, dtype)
    theta = (torch.rand(shape[1:], generator=torch.Generator().manual_seed(2)) * 0.2 - 0.02).to(DEV)
    x.view(-1)[0] = theta.view(-1)[0].to(dtype)
    g = _rand(shape, 3, 1.0, dtype)
    for bw in (1.0, 0.3):
        xr, th = x.clone().requires_grad_(), theta.clone().requires_grad_()
        y = fp8.jump_relu(xr, th, torch.tensor(bw, device=DEV) if bw < 1 else bw)
        dx, dth = torch.autograd.grad(y, (xr, th), g)
        bw = float(torch.tensor(bw))
        wy, wx, wt, mags = _jump_reference(x, theta, bw, g)
        assert torch.equal(y.double().cpu(), wy) and torch.equal(dx.double().cpu(), wx)
        assert bool(((dth.double().cpu() - wt).abs() <= (shape[0] + 4) * 2.0 ** -24 * mags).all())
    xr = x.clone().requires_grad_()
    y = fp8.jump_relu(xr)
    dx = torch.autograd.grad(y, xr, g)[0]
    assert torch.equal(y, torch.relu(x)) and torch.equal(dx, g * (x > 0))
    fp8.check_status()


def test_jump_relu_special_values():
    """Masked places may hold anything; borders of the window; zeros of both signs; NaN stays."""
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 0.53, 0.53 + 2 ** -20, -0.47, 0.03, -3.4e38, 3.4e38]], device=DEV)
    theta = torch.full((11,), 0.03, device=DEV)
    g = torch.full_like(x, 2.0)
    g[0, 1] = inf                                # no gradient where it is masked
    xr, th = x.clone().requires_grad_(), theta.clone().requires_grad_()
    y = fp8.jump_relu(xr, th, 1.0)
    dx, dth = torch.autograd.grad(y, (xr, th), g)
    wy, wx, wt, _ = _jump_reference(x, theta, 1.0, g)
    same = lambda a, b: torch.equal(torch.nan_to_num(a.double().cpu(), nan=-9.0), torch.nan_to_num(b, nan=-9.0))
    assert same(y, wy) and same(dx, wx)
    assert torch.allclose(dth.double().cpu(), wt, rtol=2 ** -22, atol=0)
    eager = x.clone().requires_grad_()
    assert torch.equal(torch.relu(x).isnan(), fp8.jump_relu(eager).isnan())


def _inside(x, theta, half):
    """theta - half < x <= theta + half exactly, in 64 bits: the rounded difference decides wherever it is not the half width itself
    (rounding keeps the order), its error (Knuth's two-sum) where it is: -0.5 + 0.5 < 1e-40, though 1e-40 + 0.5 rounds to 0.5."""
    d = x - theta
    t = d - x
    e = (x - (d - t)) + (-theta - t)
    return ((d > -half) | (d == -half) & (e > 0)) & ((d < half) | (d == half) & (e <= 0))


@pytest.mark.parametrize("as_fp32", [False, True])
@pytest.mark.parametrize("columns", [16, 15])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_jump_relu_every_16_bit_value(dtype, columns, as_fp32):
    """All 65536 values at thresholds and bandwidths up to the types' ends, aligned rows and others: results and checkpoint are
    those of the exact comparisons."""
    inf = float("inf")
    x = torch.arange(-32768, 32768).to(torch.int16).view(dtype)[:, None].expand(65536, columns).contiguous().to(DEV)
    if as_fp32:
        x = x.float()
    theta = torch.tensor([0.0, -0.5, 1e-3, 0.03, 65504.0, 1e6, -1e6, inf, float("nan"), 3.4e38, 1e-40, 2.0 ** -24, 0.53, -inf, 6e-8,
                          1.0][:columns], device=DEV)
    for bw in (1.0, 1e-6, 1e30, 1e-40, 2.0 ** -149):
        y, bits = fp8._jump_relu_forward(x, columns, theta, None, bw)
        bw = float(torch.tensor(bw))
        xd, td = x.double(), theta.double()
        want = torch.where((xd > td) & (xd > 0) | xd.isnan(), xd, torch.zeros_like(xd))
        assert torch.equal(y.double().nan_to_num(nan=-9.0), want.nan_to_num(nan=-9.0))
        words = bits.int() & 0xffff
        at = torch.arange(columns, device=DEV)
        word = words[:, at // 8]
        assert torch.equal((word >> at % 8 & 1).bool(), ~(xd < 0))
        assert torch.equal((word >> (8 + at % 8) & 1).bool(), _inside(xd, td, bw / 2))
    fp8.check_status()


@pytest.mark.parametrize("rows, columns", [(1, 24), (31, 520), (33, 2056), (129, 72), (1000, 264), (4100, 40), (515, 777)])
def test_threshold_gradient_over_the_warps_rows(rows, columns):
    """A CTA's warps share its rows: each row counts once, in the checkpoint's window, whatever the rows behind the last CTA's end."""
    for dtype in TYPES:
        x = torch.zeros(rows, columns, dtype=dtype, device=DEV).requires_grad_()
        theta = torch.ones(columns, device=DEV, requires_grad=True)
        g = (torch.arange(rows, device=DEV) % 7 + 1).to(dtype)[:, None].expand(rows, columns)
        dx, dth = torch.autograd.grad(fp8.jump_relu(x, theta, 4.0), (x, theta), g)
        assert torch.equal(dx, g)                # x = 0 passes the gradient
        assert torch.equal(dth, (-g.double().sum(0) / 4).float())    # whole numbers below 2^24: sums and a quarter are exact


def test_jump_relu_against_the_module():
    """The same results as model.JumpReLU's own autograd function."""
    from crosslayer_transcoder_b200.model import JumpReLU

    nl = JumpReLU(theta=0.03, bandwidth=0.7, n_layers=3, d_features=40).to(DEV)
    x = _rand((50, 3, 40), 1, 0.3).requires_grad_()
    g = _rand((50, 3, 40), 2)
    want = torch.autograd.grad(nl(x), (x, nl.theta), g)
    y = fp8.jump_relu(x, nl.theta, nl.bandwidth)
    got = torch.autograd.grad(y, (x, nl.theta), g)
    assert torch.equal(y, nl(x)) and torch.equal(got[0], want[0]) and got[1].shape == nl.theta.shape
    assert torch.allclose(got[1], want[1], rtol=1e-5, atol=1e-6 * float(want[1].abs().max()))


def test_jump_relu_gradient_of_x_alone():
    """Thresholds that need no gradient change nothing for x; so do they for many short rows."""
    x, th, g = _rand((500, 40), 1, 0.2), torch.full((40,), 0.05, device=DEV), _rand((500, 40), 2)
    xr, tr = x.clone().requires_grad_(), th.clone().requires_grad_()
    want = torch.autograd.grad(fp8.jump_relu(xr, tr, 0.5), (xr, tr), g)
    assert torch.equal(torch.autograd.grad(fp8.jump_relu(xr, th, 0.5), xr, g)[0], want[0])
    assert torch.equal(torch.autograd.grad(fp8.jump_relu(x, tr, 0.5), tr, g)[0], want[1])
    long = torch.randn(9_000_000, 8, device=DEV)
    assert torch.equal(fp8.jump_relu(long), torch.relu(long))


def test_jump_relu_strides_and_empty():
    base = _rand((30, 4, 100), 1)
    for x in (base[:, 1], base[:, :, 3:50], base[::2], base[:, 0].t(), base[0, 0].expand(9, 100), base[:0]):
        assert torch.equal(fp8.jump_relu(x), torch.relu(x))
    x = base[:0].clone().requires_grad_()
    th = torch.zeros(4, 100, device=DEV, requires_grad=True)
    dx, dth = torch.autograd.grad(fp8.jump_relu(x, th), (x, th), torch.zeros_like(x))
    assert dx.shape == x.shape and not dth.any()
    x = base.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(fp8.jump_relu(x).sum(), x)[0], (base > 0).float())
