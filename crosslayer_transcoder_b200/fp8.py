"""8-bit operands and checkpoints: block-scaled e4m3 copies of activations and weights, their products on the tensor cores, and
the transcoder's differentiable passes built from them.

    q = quantize(x)                          BlockTensor: e4m3 values with a scale for each block of 128 x 128 (or 1 x 128)
    y = matmul(a, b, bias)                   product of two of them, fp32 sums
    y = project(x, W, b)                     Encoder.forward, Decoder.forward (per-layer)     } differentiable; what is kept for
    y = crosslayer_decode(f, blocks, b)      CrosslayerDecoder.forward                        } backward are the 8-bit operands
    f = jump_relu(pre, theta, bandwidth)     JumpReLU / ReLU; what is kept are two bits an element

A product takes its operands as the 8-bit values stand for them and rounds its fp32 sums once.  ``project`` and
``crosslayer_decode`` quantise the input, the weights and the incoming gradient by blocks of 128 x 128, so that one copy serves the
products along either of its axes: the input's copy is the forward operand and the checkpoint of the weight gradient.  Their
gradients are those of the products with the operands as they stand (straight through the rounding); the bias gets the sum of
the gradient as it came in.  Rounding an element to e4m3 moves it by up to 2^-4 of its value (with the block's largest
magnitude at 224 to 448, elements below 2^-18 of it become 0).

``CrossLayerTranscoder.eight_bit = True`` runs the model's forward on these (``crosslayer_transcoder_b200.model.clt``).

Everything is enqueued on the current stream of the operands' device; scratch is torch's.  The kernels report a failure in a
status word in host memory, which every call looks at: ``CltError`` is raised by a later call, or by ``check_status()``, which
waits for the device first.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import DTYPE_CODE, CltError, lib, stream_ptr

__all__ = ["BlockTensor", "quantize", "matmul", "project", "crosslayer_decode", "jump_relu", "check_status"]

BLOCK = 128
_BATCHED, _DEC_FWD, _DEC_DFEAT, _DEC_DW = range(4)

_status: Optional[torch.Tensor] = None       # one pinned word for all devices; kernels write to it only when they fail
_status_view = None


def _blocks(n: int, rows: int = BLOCK) -> int:
    return -(-n // rows)


def _status_word() -> torch.Tensor:
    global _status, _status_view
    if _status is None:
        if torch.cuda.is_current_stream_capturing():
            raise CltError("make one 8-bit call before a graph is captured: the first one allocates its status word")
        word = torch.zeros(1, dtype=torch.int32).pin_memory()
        _status, _status_view = word, word.numpy()
    if _status_view[0] != 0:
        _raise_status("(reported by an earlier call)")
    return _status


def _raise_status(where: str):
    code, _status_view[0] = int(_status_view[0]), 0
    raise CltError(f"device status {code:#x} {where}: {_lib.STATUS_NAMES.get(code, 'unknown code')}")


def check_status(where: str = ""):
    """Wait for the current device and raise ``CltError`` if a kernel of an 8-bit call gave up."""
    if _status is not None:
        torch.cuda.synchronize()
        if _status_view[0] != 0:
            _raise_status(where)


def _need(cond: bool, text: str):
    if not cond:
        raise ValueError(text)


def _check(name: str, t, dtypes=None, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")


class _On:
    """The device of the operands as the current one."""

    def __init__(self, device):
        if device.type != "cuda":
            raise CltError(f"the 8-bit operators run on CUDA tensors only (no CPU fallback), got {device}")
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        lib().check_device()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _storage(*shape, device):
    """8-bit values [..., C] whose rows start on 16 bytes."""
    pitch = -(-shape[-1] // 16) * 16
    return torch.empty(*shape[:-1], pitch, dtype=torch.float8_e4m3fn, device=device)[..., :shape[-1]]


class BlockTensor:
    """e4m3 ``values [R, C]`` or ``[Z, R, C]`` with fp32 ``scales [(Z,) ceil(R / block_rows), ceil(C / 128)]``: an element stands
    for its value times the scale of its block, the blocks being ``block_rows`` (1 or 128) x 128 from the matrix's origin on.
    ``scales`` may be any fp32 numbers; ``quantize`` makes powers of two."""

    __slots__ = ("values", "scales", "block_rows", "transposed")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, block_rows: int = BLOCK):
        _check("values", values, (torch.float8_e4m3fn,))
        _check("scales", scales, (torch.float32,), values.device)
        _need(block_rows in (1, BLOCK), f"blocks of {block_rows} rows: 1 or 128 are supported")
        _need(values.dim() in (2, 3), f"expected a matrix or a stack of matrices, got {tuple(values.shape)}")
        want = (*values.shape[:-2], _blocks(values.shape[-2], block_rows), _blocks(values.shape[-1]))
        _need(tuple(scales.shape) == want, f"scales {tuple(scales.shape)} do not match {want}")
        self.values, self.scales, self.block_rows, self.transposed = values, scales, block_rows, False

    @property
    def shape(self) -> torch.Size:
        s = self.values.shape
        return torch.Size((*s[:-2], s[-1], s[-2])) if self.transposed else s

    @property
    def device(self):
        return self.values.device

    @property
    def mT(self) -> "BlockTensor":
        """The transposed matrices, without a copy."""
        t = BlockTensor(self.values, self.scales, self.block_rows)
        t.transposed = not self.transposed
        return t

    def __getitem__(self, i: int) -> "BlockTensor":
        _need(self.values.dim() == 3, "only a stack of matrices is indexed")
        t = BlockTensor(self.values[i], self.scales[i], self.block_rows)
        t.transposed = self.transposed
        return t

    def __repr__(self):
        return f"BlockTensor(shape={tuple(self.shape)}, block_rows={self.block_rows}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the elements stand for, rounded once to ``dtype`` (fp32, fp16 or bf16)."""
        _need(dtype in DTYPE_CODE, f"dequantize to fp32, fp16 or bf16, not {dtype}")
        v, s = self._stack()
        Z, R, C = v.shape
        with _On(self.device):
            out = torch.empty(Z, R, C, dtype=dtype, device=self.device)
            if out.numel():
                if v.stride(2) != 1:
                    v = v.contiguous()
                lib().call("clt_fp8_dequantize", v, v.stride(1), v.stride(0), s, *s.stride(), self.block_rows, out,
                           DTYPE_CODE[dtype], Z, R, C, stream_ptr())
        out = out.view(self.values.shape)
        return out.mT if self.transposed else out

    def _stack(self):
        v, s = self.values, self.scales
        return (v, s) if v.dim() == 3 else (v.unsqueeze(0), s.unsqueeze(0))


def _quantize(x: torch.Tensor, block_rows: int, sums: bool = False, into=None):
    """(values, scales, column sums of x or None) of x [Z, R, C]; ``into``: (values, scales) to write to."""
    if x.stride(2) != 1 and x.shape[2] > 1:
        x = x.contiguous()
    Z, R, C = x.shape
    v, s = into or (_storage(Z, R, C, device=x.device),
                    torch.empty(Z, _blocks(R, block_rows), _blocks(C), dtype=torch.float32, device=x.device))
    part = torch.empty(Z, _blocks(R), C, dtype=torch.float32, device=x.device) if sums else None
    total = torch.empty(Z, C, dtype=torch.float32, device=x.device) if sums else None
    if x.numel():
        lib().call("clt_fp8_quantize", x, DTYPE_CODE[x.dtype], x.stride(1), x.stride(0), v, v.stride(1), s, part, Z, R, C,
                   block_rows, stream_ptr())
        if sums:
            lib().call("clt_sum_chunks", part, total, Z, _blocks(R), C, stream_ptr())
    elif sums:
        total.zero_()
    return v, s, total


def quantize(x: torch.Tensor, block_rows: int = BLOCK) -> BlockTensor:
    """``x [R, C]`` or ``[Z, R, C]`` (fp32, fp16 or bf16) in 8 bits.  A block's scale is the smallest power of two (at least 2^-126)
    that brings its largest finite magnitude to at most 448, the largest e4m3 value; 1 for a block of zeros.  Elements are rounded
    to nearest; what is not finite becomes NaN and does not count for the scale."""
    _check("x", x, DTYPE_CODE)
    _need(x.dim() in (2, 3), f"expected a matrix or a stack of matrices, got {tuple(x.shape)}")
    _need(block_rows in (1, BLOCK), f"blocks of {block_rows} rows: 1 or 128 are supported")
    x = x.detach()
    with _On(x.device):
        v, s, _ = _quantize(x if x.dim() == 3 else x.unsqueeze(0), block_rows)
    return BlockTensor(v, s, block_rows) if x.dim() == 3 else BlockTensor(v[0], s[0], block_rows)


# ---- products ----------------------------------------------------------------------------------------------------------------
def _aligned(v: torch.Tensor) -> torch.Tensor:
    """``v [Z, R, C]``, copied where the tensor-core path cannot read it in place: rows have to start on 16 bytes."""
    Z, R, C = v.shape
    if (v.stride(2) == 1 or C == 1) and v.data_ptr() % 16 == 0 and (R == 1 or (v.stride(1) % 16 == 0 and v.stride(1) >= C)) and \
            (Z == 1 or (v.stride(0) % 16 == 0 and v.stride(0) > 0)):
        return v
    out = _storage(Z, R, C, device=v.device)
    out.view(torch.uint8).copy_(v.view(torch.uint8))
    return out


def _operand(v: torch.Tensor, s: torch.Tensor, transposed: bool, along_k_is_row: bool):
    """(values, row distance, matrix distance, transposed, scales and their distances: matrices, along M or N, along K)."""
    Z, R, C = v.shape
    ld = v.stride(1) if R > 1 else -(-C // 16) * 16
    sz, sr, sc = s.stride()
    mn, k = (sc, sr) if along_k_is_row else (sr, sc)
    return (v, ld, v.stride(0), int(transposed), s, sz, mn, k)


def _contract(mode: int, a, a_t: bool, b, b_t: bool, bias, out: torch.Tensor, out_ld: int, out_z: int, M: int, N: int, K: int,
              L: int, a_rows: int = BLOCK):
    """One call of the contraction.  ``a``, ``b``: (values [*, R, C], scales); ``a_t``: A is stored [K, M]; ``b_t``: B [N, K]."""
    status = _status_word()
    parts = lib().query("clt_fp8_matmul_parts", mode, M, N, K, L, 0)
    ws = torch.empty(parts * M * N, dtype=torch.float32, device=out.device) if parts else None
    lib().call("clt_fp8_matmul", mode, *_operand(*a, a_t, a_t), a_rows, *_operand(*b, b_t, not b_t), bias,
               bias.stride(0) if bias is not None else 0, out, DTYPE_CODE[out.dtype], out_ld, out_z, ws, parts * M * N, M, N, K, L,
               status, stream_ptr())


def matmul(a: BlockTensor, b: BlockTensor, bias: Optional[torch.Tensor] = None,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a [M, K] @ b [K, N] (+ bias [N])``, or stacks ``[Z, M, K] @ [Z, K, N] (+ bias [N] or [Z, N])``, in fp32 sums that are
    rounded once to ``out_dtype``.  ``a`` has blocks of 1 x 128 or 128 x 128 (with 1 x 128 only untransposed: its blocks have to
    lie along the contraction), ``b`` blocks of 128 x 128; either may be a transposed view (``.mT``).  The products of the
    operands' scales have to be finite.  Values whose rows do not start on 16 bytes are copied first."""
    for name, t in (("a", a), ("b", b)):
        if not isinstance(t, BlockTensor):
            raise TypeError(f"{name} must be a BlockTensor, got {type(t).__name__}")
    _need(a.values.dim() == b.values.dim(), f"a {tuple(a.shape)} and b {tuple(b.shape)} must both be matrices or both stacks")
    _need(a.device == b.device, f"a is on {a.device}, b on {b.device}")
    _need(a.shape[-1] == b.shape[-2] and a.shape[:-2] == b.shape[:-2], f"a {tuple(a.shape)} does not match b {tuple(b.shape)}")
    _need(b.block_rows == BLOCK, "b needs blocks of 128 x 128")
    _need(a.block_rows == BLOCK or not a.transposed, "a transposed operand needs blocks of 128 x 128")
    _need(out_dtype in DTYPE_CODE, f"the result is fp32, fp16 or bf16, not {out_dtype}")
    (va, sa), (vb, sb) = a._stack(), b._stack()
    Z, M, K, N = va.shape[0], a.shape[-2], a.shape[-1], b.shape[-1]
    if bias is not None:
        _check("bias", bias, DTYPE_CODE, a.device)
        _need(tuple(bias.shape) in ((N,), (Z, N)), f"bias {tuple(bias.shape)} does not match {(Z, N)}")
        bias = bias.detach().float().expand(Z, N)
        if bias.stride(1) != 1 and N > 1:
            bias = bias.contiguous()
    with _On(a.device):
        out = torch.empty(*a.shape[:-1], N, dtype=out_dtype, device=a.device)
        if out.numel() == 0:
            return out
        if K == 0:
            return out.zero_() if bias is None else out.copy_(bias.unsqueeze(1).expand(Z, M, N).view(out.shape))
        _contract(_BATCHED, (_aligned(va), sa), a.transposed, (_aligned(vb), sb), b.transposed, bias, out, N, M * N, M, N, K, Z,
                  a.block_rows)
    return out


# ---- differentiable passes ------------------------------------------------------------------------------------------------------
def _bias32(b):
    return None if b is None else b.detach().float().contiguous()


class _Project(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, W, b):
        B, L, D = x.shape
        F = W.shape[2]
        ctx.dims, ctx.types = (B, L, D, F), (x.dtype, W.dtype, None if b is None else b.dtype)
        with _On(x.device):
            y = torch.empty(B, L, F, dtype=x.dtype, device=x.device)
            xv, xs, _ = _quantize(x.transpose(0, 1), BLOCK)
            wv, ws, _ = _quantize(W, BLOCK)
            if B:
                _contract(_BATCHED, (xv, xs), False, (wv, ws), False, _bias32(b), y, L * F, F, B, F, D, L)
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.save_for_backward(*((xv, xs) if need_w else (None, None)), *((wv, ws) if need_x else (None, None)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        xv, xs, wv, ws = ctx.saved_tensors
        B, L, D, F = ctx.dims
        dx = dW = db = None
        need_x, need_w, need_b = ctx.needs_input_grad
        with _On(g.device):
            gv, gs, db = _quantize(g.transpose(0, 1), BLOCK, sums=need_b)
            if need_x:
                dx = torch.empty(B, L, D, dtype=ctx.types[0], device=g.device)
                if B:
                    _contract(_BATCHED, (gv, gs), False, (wv, ws), True, None, dx, L * D, D, B, D, F, L)
            if need_w:
                dW = torch.empty(L, D, F, dtype=ctx.types[1], device=g.device)
                if B:
                    _contract(_BATCHED, (xv, xs), True, (gv, gs), False, None, dW, F, D * F, D, F, B, L)
                else:
                    dW.zero_()
        return dx, dW, db.to(ctx.types[2]) if need_b else None


def project(x: torch.Tensor, W: torch.Tensor, b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., L, D] -> [..., L, F]`` by layer ``l``'s ``W[l] [D, F]`` (and ``b [L, F]``), as ``Encoder.forward`` and the
    per-layer ``Decoder.forward``; or ``x [..., D]`` by one ``W [D, F]`` (and ``b [F]``).  Operands in 8 bits, result in ``x``'s type.
    Differentiable in ``x``, ``W`` and ``b``: backward reads the 8-bit copies of ``x`` and ``W`` that forward made and quantises
    the incoming gradient; one call keeps ``B L D + L D F`` bytes."""
    _check("x", x, DTYPE_CODE)
    _check("W", W, DTYPE_CODE, x.device)
    _need(W.dim() in (2, 3), f"expected W [D, F] or [L, D, F], got {tuple(W.shape)}")
    one = W.dim() == 2
    inner = tuple(W.shape[:2]) if not one else (W.shape[0],)
    _need(x.dim() > len(inner) - 1 and tuple(x.shape[x.dim() - len(inner):]) == inner, f"x {tuple(x.shape)} does not match W {tuple(W.shape)}")
    _need(W.numel() > 0, f"empty W {tuple(W.shape)}")
    if b is not None:
        _check("b", b, DTYPE_CODE, x.device)
        _need(tuple(b.shape) == (W.shape[-1],) if one else tuple(b.shape) == (W.shape[0], W.shape[2]),
              f"b {tuple(b.shape)} does not match W {tuple(W.shape)}")
    lead = x.shape[:x.dim() - len(inner)]
    if one:
        W, b = W.unsqueeze(0), None if b is None else b.unsqueeze(0)
    y = _Project.apply(x.reshape(lead.numel(), *W.shape[:2]), W, b)
    return y.view(*lead, *((W.shape[2],) if one else (W.shape[0], W.shape[2])))


class _CrosslayerDecode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, b, *blocks):
        B, L, F = f.shape
        D = blocks[0].shape[2]
        P = L * (L + 1) // 2
        ctx.dims, ctx.types = (B, L, F, D), (f.dtype, None if b is None else b.dtype, [w.dtype for w in blocks])
        with _On(f.device):
            y = torch.empty(B, L, D, dtype=f.dtype, device=f.device)
            fv, fs, _ = _quantize(f.transpose(0, 1), BLOCK)
            wv = _storage(P, F, D, device=f.device)
            ws = torch.empty(P, _blocks(F), _blocks(D), dtype=torch.float32, device=f.device)
            for t, w in enumerate(blocks):
                at = slice(t * (t + 1) // 2, (t + 1) * (t + 2) // 2)
                _quantize(w, BLOCK, into=(wv[at], ws[at]))
            if B:
                _contract(_DEC_FWD, (fv, fs), False, (wv, ws), False, _bias32(b), y, L * D, D, B, D, F, L)
        need_f, need_w = ctx.needs_input_grad[0], any(ctx.needs_input_grad[2:])
        ctx.save_for_backward(*((fv, fs) if need_w else (None, None)), *((wv, ws) if need_f else (None, None)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        fv, fs, wv, ws = ctx.saved_tensors
        B, L, F, D = ctx.dims
        df = db = None
        need_f, need_b, *need_w = ctx.needs_input_grad
        dW = [None] * L
        with _On(g.device):
            gv, gs, db = _quantize(g.transpose(0, 1), BLOCK, sums=need_b)
            if need_f:
                df = torch.empty(B, L, F, dtype=ctx.types[0], device=g.device)
                if B:
                    _contract(_DEC_DFEAT, (gv, gs), False, (wv, ws), True, None, df, L * F, F, B, F, D, L)
            if any(need_w):
                P = L * (L + 1) // 2
                flat = torch.empty(P, F, D, dtype=torch.float32, device=g.device)
                if B:
                    _contract(_DEC_DW, (fv, fs), True, (gv, gs), False, None, flat, D, F * D, F, D, B, L)
                else:
                    flat.zero_()
                dW = [flat[t * (t + 1) // 2:(t + 1) * (t + 2) // 2].to(ctx.types[2][t]) if need_w[t] else None for t in range(L)]
        return (df, db.to(ctx.types[1]) if need_b else None, *dW)


def crosslayer_decode(features: torch.Tensor, blocks: Sequence[torch.Tensor], b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``features [..., L, F] -> [..., L, D]``: target layer ``t`` gets ``sum over s <= t of features[..., s, :] @ blocks[t][s]`` (and
    ``b[t]``), ``blocks[t]`` being ``[t + 1, F, D]``, as ``CrosslayerDecoder.forward``.  Types, rounding and what is kept for backward as
    in ``project``: ``B L F + P F D`` bytes for the P blocks of the decoder."""
    _check("features", features, DTYPE_CODE)
    _need(features.dim() >= 2, f"expected features [..., L, F], got {tuple(features.shape)}")
    L, F = features.shape[-2:]
    blocks = list(blocks)
    _need(L > 0 and len(blocks) == L, f"{len(blocks)} decoder blocks for {L} layers")
    for t, w in enumerate(blocks):
        _check(f"blocks[{t}]", w, DTYPE_CODE, features.device)
        _need(w.dim() == 3 and w.shape[:2] == (t + 1, F) and w.shape[2] == blocks[0].shape[2],
              f"blocks[{t}] {tuple(w.shape)} does not match {(t + 1, F, blocks[0].shape[-1])}")
    D = blocks[0].shape[2]
    _need(F > 0 and D > 0, f"empty decoder blocks {tuple(blocks[0].shape)}")
    if b is not None:
        _check("b", b, DTYPE_CODE, features.device)
        _need(tuple(b.shape) == (L, D), f"b {tuple(b.shape)} does not match {(L, D)}")
    lead = features.shape[:-2]
    return _CrosslayerDecode.apply(features.reshape(lead.numel(), L, F), b, *blocks).view(*lead, L, D)


class _JumpReLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, theta, bandwidth):
        R, C = x.shape
        on_device = isinstance(bandwidth, torch.Tensor)
        ctx.bandwidth = 0.0 if on_device else float(bandwidth)
        with _On(x.device):
            if x.stride(1) != 1 and C > 1:
                x = x.contiguous()
            y = torch.empty(R, C, dtype=x.dtype, device=x.device)
            bits = torch.empty(R, -(-C // 8), dtype=torch.int16, device=x.device)
            th = None if theta is None else theta.detach().float().contiguous()
            bw = bandwidth.detach().float() if on_device else None
            if y.numel():
                lib().call("clt_jump_relu_fwd", x, x.stride(0), th, bw, ctx.bandwidth, y, bits, DTYPE_CODE[x.dtype], R, C, stream_ptr())
        ctx.theta_type = None if theta is None else theta.dtype
        ctx.save_for_backward(bits, th, bw)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        bits, th, bw = ctx.saved_tensors
        R, C = g.shape
        if g.stride(1) != 1 and C > 1:
            g = g.contiguous()
        dx = torch.empty(R, C, dtype=g.dtype, device=g.device)
        dth = None if th is None else torch.zeros(C, dtype=torch.float32, device=g.device) if R == 0 else \
            torch.empty(C, dtype=torch.float32, device=g.device)
        with _On(g.device):
            if dx.numel():
                n = lib().query("clt_jump_relu_chunks", R, C) * C if th is not None else 0
                ws = torch.empty(n, dtype=torch.float32, device=g.device) if n else None
                lib().call("clt_jump_relu_bwd", g, g.stride(0), bits, th, bw, ctx.bandwidth, dx, dth, ws, n, DTYPE_CODE[g.dtype], R, C,
                           stream_ptr())
        return dx, None if dth is None else dth.to(ctx.theta_type), None


def jump_relu(x: torch.Tensor, theta: Optional[torch.Tensor] = None, bandwidth=1.0) -> torch.Tensor:
    """JumpReLU ``x [x > theta and x > 0]`` with the thresholds ``theta`` (``x``'s last axes, e.g. ``[L, F]`` or ``[1, L, F]``
    for ``x [..., L, F]``), or ReLU without.  Differentiable in ``x`` and ``theta`` as ``model.JumpReLU``: ``dx = g [x >= 0]`` (ReLU:
    ``[x > 0]``), ``dtheta = -(theta / bandwidth) sum g [theta - bandwidth / 2 < x <= theta + bandwidth / 2]``, from two bits an
    element instead of ``x``.  A masked element is 0 and gets no gradient whatever it was; NaN stays NaN.  ``bandwidth``: a positive number,
    or one on ``x``'s device."""
    _check("x", x, DTYPE_CODE)
    shape = x.shape
    _need(x.dim() >= 1, "x has no axis")
    if theta is None:
        C = shape[-1]
        flat = None
    else:
        _check("theta", theta, DTYPE_CODE, x.device)
        inner = tuple(theta.shape)
        while len(inner) > 1 and inner[0] == 1 and inner != tuple(shape[len(shape) - len(inner):]):
            inner = inner[1:]
        _need(len(inner) >= 1 and len(inner) <= len(shape) and tuple(shape[len(shape) - len(inner):]) == inner,
              f"theta {tuple(theta.shape)} does not match the last axes of x {tuple(shape)}")
        C = theta.numel()
        flat = theta.reshape(C)
        if isinstance(bandwidth, torch.Tensor):
            _check("bandwidth", bandwidth, DTYPE_CODE, x.device)
            _need(bandwidth.numel() == 1, f"bandwidth has {bandwidth.numel()} elements")
        else:
            _need(float(bandwidth) > 0, f"bandwidth must be positive, got {bandwidth}")
    rows = x.numel() // C if C else 0
    return _JumpReLU.apply(x.reshape(rows, C), flat, bandwidth).view(shape)
