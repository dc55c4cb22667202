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

import threading
from array import array
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
_status_lock = threading.Lock()


def _blocks(n: int, rows: int = BLOCK) -> int:
    return -(-n // rows)


def _status_word() -> torch.Tensor:
    global _status, _status_view
    if _status is None:
        if torch.cuda.is_current_stream_capturing():
            raise CltError("make one 8-bit call before a graph is captured: the first one allocates its status word")
        with _status_lock:
            if _status is None:
                word = torch.zeros(1, dtype=torch.int32).pin_memory()
                _status_view = word.numpy()
                _status = word
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


def _check(name: str, t, dtypes, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


MOST = 2 ** 31 - 256    # rows or columns of a matrix: the kernels count them, rounded up to tiles, in 32 bits


def _fits(name: str, *sizes: int):
    if max(sizes) > MOST:
        raise ValueError(f"{name} has {' x '.join(map(str, sizes))} elements, at most {MOST} along an axis are supported")


_checked = set()        # devices that the library runs on


def _on(device, fn, *args):
    """``fn(*args)`` with the operands' device as the current one."""
    if device.index in _checked and device.type == "cuda" and torch._C._cuda_getDevice() == device.index:
        return fn(*args)
    if device.type != "cuda":
        raise CltError(f"the 8-bit operators run on CUDA tensors only (no CPU fallback), got {device}")
    with torch.cuda.device(device):
        lib().check_device()
        _checked.add(device.index)
        return fn(*args)


def _first_order(backward):
    """``once_differentiable``, whose wrapper is entered only where a graph of the gradient is asked for."""
    once = once_differentiable(backward)
    return lambda ctx, g: once(ctx, g) if torch.is_grad_enabled() else backward(ctx, g)


def _pitch(C: int) -> int:
    """Bytes from row to row of a copy.  16 are enough for the contraction; rows that start on a memory sector are written faster
    (12 x 4000 x 10000 bf16: 244 -> 225 us)."""
    return (C + 31) & ~31


def _storage(*shape, device):
    """8-bit values [..., C] whose rows start on 32 bytes."""
    C = shape[-1]
    v = torch.empty(*shape[:-1], _pitch(C), dtype=torch.float8_e4m3fn, device=device)
    return v if C % 32 == 0 else v[..., :C]


class BlockTensor:
    """e4m3 ``values [R, C]`` or ``[Z, R, C]`` with fp32 ``scales [(Z,) ceil(R / block_rows), ceil(C / 128)]``: an element stands
    for its value times the scale of its block, the blocks being ``block_rows`` (1 or 128) x 128 from the matrix's origin on.
    ``scales`` may be any fp32 numbers; ``quantize`` makes powers of two."""

    __slots__ = ("values", "scales", "block_rows", "transposed")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, block_rows: int = BLOCK):
        _check("values", values, (torch.float8_e4m3fn,))
        _check("scales", scales, (torch.float32,), values.device)
        if block_rows not in (1, BLOCK):
            raise ValueError(f"blocks of {block_rows} rows: 1 or 128 are supported")
        shape = values.shape
        if len(shape) not in (2, 3):
            raise ValueError(f"expected a matrix or a stack of matrices, got {tuple(shape)}")
        want = (*shape[:-2], _blocks(shape[-2], block_rows), _blocks(shape[-1]))
        if scales.shape != want:
            raise ValueError(f"scales {tuple(scales.shape)} do not match {want}")
        _fits("values", *shape)
        self.values, self.scales, self.block_rows, self.transposed = values, scales, block_rows, False

    @classmethod
    def _of(cls, values, scales, block_rows, transposed=False):
        t = object.__new__(cls)
        t.values, t.scales, t.block_rows, t.transposed = values, scales, block_rows, transposed
        return t

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
        return self._of(self.values, self.scales, self.block_rows, not self.transposed)

    def __getitem__(self, i: int) -> "BlockTensor":
        if self.values.dim() != 3 or type(i) is not int:     # (True would add an axis)
            raise ValueError("a stack of matrices is indexed with one integer")
        return self._of(self.values[i], self.scales[i], self.block_rows, self.transposed)

    def __repr__(self):
        return f"BlockTensor(shape={tuple(self.shape)}, block_rows={self.block_rows}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """What the elements stand for, rounded once to ``dtype`` (fp32, fp16 or bf16)."""
        if dtype not in DTYPE_CODE:
            raise ValueError(f"dequantize to fp32, fp16 or bf16, not {dtype}")
        out = _on(self.device, _dequantize, self.values, self.scales, self.block_rows, dtype)
        return out.mT if self.transposed else out


def _dequantize(v, s, block_rows, dtype):
    out = torch.empty(v.shape, dtype=dtype, device=v.device)
    if out.numel():
        if v.stride(-1) != 1:
            v = v.contiguous()
        Z, v_z, s_z = (v.shape[0], v.stride(0), s.stride(0)) if v.dim() == 3 else (1, 0, 0)
        R, C = v.shape[-2:]
        lib().call("clt_fp8_dequantize", v, v.stride(-2), v_z, s, s_z, s.stride(-2), s.stride(-1), block_rows, out,
                   DTYPE_CODE[dtype], Z, R, C, stream_ptr())
    return out


def _quantize_any(x, block_rows):
    """quantize of a matrix or a stack."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    shape = x.shape
    R, C = shape[-2:]
    Z, x_z = (shape[0], x.stride(0)) if len(shape) == 3 else (1, 0)
    v = _storage(*shape, device=x.device)
    s = torch.empty(*shape[:-2], _blocks(R, block_rows), _blocks(C), dtype=torch.float32, device=x.device)
    if x.numel():
        lib().call("clt_fp8_quantize", x, DTYPE_CODE[x.dtype], x.stride(-2), x_z, v, _pitch(C), s, None, Z, R, C, block_rows,
                   stream_ptr())
    return BlockTensor._of(v, s, block_rows)


def quantize(x: torch.Tensor, block_rows: int = BLOCK) -> BlockTensor:
    """``x [R, C]`` or ``[Z, R, C]`` (fp32, fp16 or bf16) in 8 bits.  A block's scale is the smallest power of two (at least 2^-126)
    that brings its largest finite magnitude to at most 448, the largest e4m3 value; 1 for a block of zeros.  Elements are rounded
    to nearest; what is not finite becomes NaN and does not count for the scale."""
    _check("x", x, DTYPE_CODE)
    if x.dim() not in (2, 3):
        raise ValueError(f"expected a matrix or a stack of matrices, got {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"blocks of {block_rows} rows: 1 or 128 are supported")
    _fits("x", *x.shape)
    return _on(x.device, _quantize_any, x.detach(), block_rows)


# ---- products ----------------------------------------------------------------------------------------------------------------
def _operand(v: torch.Tensor, s: torch.Tensor, rows_are_k: bool, transposed: bool):
    """What ``clt_fp8_matmul`` takes of an operand: values, distances of rows and matrices, whether it is stored transposed, scales and
    their distances between matrices, along M or N and along K.  Copied where the tensor-core path cannot read the values in place:
    rows have to start on 16 bytes."""
    stack = v.dim() == 3
    Z, z = (v.shape[0], v.stride(0)) if stack else (1, 0)
    R, C = v.shape[-2:]
    ld = v.stride(-2)
    if R == 1:
        ld = _pitch(C)
    if (v.stride(-1) != 1 and C > 1) or ld % 16 or ld < C or v.data_ptr() % 16 or (Z > 1 and (z % 16 or z <= 0)):
        if v.stride(-1) != 1 and C > 1:
            v = v.contiguous()
            z = v.stride(0) if stack else 0
        copy = torch.empty(*v.shape[:-1], _pitch(C), dtype=torch.uint8, device=v.device)
        lib().call("clt_fp8_align", v, v.stride(-2), z, copy, _pitch(C), Z, R, C, stream_ptr())
        v, ld, z = copy, _pitch(C), R * _pitch(C)
    sr, sc = s.stride(-2), s.stride(-1)
    return v, ld, z, int(transposed), s, s.stride(0) if stack else 0, *((sc, sr) if rows_are_k else (sr, sc))


def _contract(mode: int, a, b, bias, bias_z: int, out, out_ld: int, out_z: int, M: int, N: int, K: int, L: int,
              a_rows: int = BLOCK):
    """One call of the contraction.  ``a``, ``b``: as ``_operand`` describes them."""
    status = _status_word()
    parts = lib().query("clt_fp8_matmul_parts", mode, M, N, K, L, 0)
    ws = torch.empty(parts * M * N, dtype=torch.float32, device=out.device) if parts else None
    lib().call("clt_fp8_matmul", mode, *a, a_rows, *b, bias, bias_z, out, DTYPE_CODE[out.dtype], out_ld, out_z, ws, parts * M * N,
               M, N, K, L, status, stream_ptr())


def _matmul(a, b, bias, out_dtype):
    va, vb = a.values, b.values
    M, K = va.shape[-2:] if not a.transposed else (va.shape[-1], va.shape[-2])
    N = vb.shape[-2] if b.transposed else vb.shape[-1]
    Z = va.shape[0] if va.dim() == 3 else 1
    out = torch.empty(*va.shape[:-2], M, N, dtype=out_dtype, device=va.device)
    if out.numel() == 0:
        return out
    bias_z = 0
    if bias is not None:
        bias = bias.detach()
        if bias.dtype != torch.float32 or bias.stride(-1) != 1:
            bias = bias.float().contiguous()
        bias_z = bias.stride(0) if bias.dim() == 2 else 0
    if K == 0:
        return out.zero_() if bias is None else out.copy_(bias.unsqueeze(-2).expand(out.shape) if bias.dim() == va.dim() - 1
                                                           else bias.expand(out.shape))
    _contract(_BATCHED, _operand(va, a.scales, a.transposed, a.transposed), _operand(vb, b.scales, not b.transposed, b.transposed),
              bias, bias_z, out, N, M * N, M, N, K, Z, a.block_rows)
    return out


def matmul(a: BlockTensor, b: BlockTensor, bias: Optional[torch.Tensor] = None,
           out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``a [M, K] @ b [K, N] (+ bias [N])``, or stacks ``[Z, M, K] @ [Z, K, N] (+ bias [N] or [Z, N])``, in fp32 sums that are
    rounded once to ``out_dtype``.  ``a`` has blocks of 1 x 128 or 128 x 128 (with 1 x 128 only untransposed: its blocks have to
    lie along the contraction), ``b`` blocks of 128 x 128; either may be a transposed view (``.mT``).  Values whose rows do not start on 16 bytes are copied first."""
    if not isinstance(a, BlockTensor) or not isinstance(b, BlockTensor):
        raise TypeError(f"a and b must be BlockTensors, got {type(a).__name__} and {type(b).__name__}")
    sa, sb = a.shape, b.shape
    if len(sa) != len(sb):
        raise ValueError(f"a {tuple(sa)} and b {tuple(sb)} must both be matrices or both stacks")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device}, b on {b.device}")
    if sa[-1] != sb[-2] or (len(sa) == 3 and sa[0] != sb[0]):
        raise ValueError(f"a {tuple(sa)} does not match b {tuple(sb)}")
    if b.block_rows != BLOCK:
        raise ValueError("b needs blocks of 128 x 128")
    if a.block_rows != BLOCK and a.transposed:
        raise ValueError("a transposed operand needs blocks of 128 x 128")
    if out_dtype not in DTYPE_CODE:
        raise ValueError(f"the result is fp32, fp16 or bf16, not {out_dtype}")
    if bias is not None:
        _check("bias", bias, DTYPE_CODE, a.device)
        if bias.shape != sb[-1:] and (len(sb) != 3 or bias.shape != (sb[0], sb[2])):
            raise ValueError(f"bias {tuple(bias.shape)} does not match b {tuple(sb)}")
    return _on(a.device, _matmul, a, b, bias, out_dtype)


# ---- differentiable passes ------------------------------------------------------------------------------------------------------
_BYTES = dict(dtype=torch.uint8)


def _rows_first(x):
    """x [B, L, C] with unit distance inside a row: (x, distance of rows, distance of layers)."""
    if x.is_contiguous():
        return x, x.shape[1] * x.shape[2], x.shape[2]
    if x.stride(2) != 1 and x.shape[2] > 1:
        x = x.contiguous()
    return x, x.stride(0), x.stride(1)


def _pass_forward(crosslayer, x, W, blocks, w_dtype, b, shape):
    """y [B, L, N] as ``shape`` and the 8-bit copies of x [B, L, K] and of the weights (``W``, or the addresses of a decoder's
    ``blocks``).  (y is made in its final shape: of a view that a node returns autograd refuses changes in place.)"""
    status, call, query, dev = _status_word(), lib().call, lib().query, x.device
    (B, L, K), N = x.shape, shape[-1]
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    x_copy = torch.empty(256 * query("clt_fp8_copy_units", L, B, K), device=dev, **_BYTES)
    w_copy = torch.empty(256 * query("clt_fp8_copy_units", _pairs(L) if crosslayer else L, K, N), device=dev, **_BYTES)
    if B:
        n = query("clt_fp8_pass_units", crosslayer, 0, 0, 0, 0, B, L, K, N)
        scratch = torch.empty(256 * n, device=dev, **_BYTES) if n else None
        x, ld, z = _rows_first(x)
        if b is not None and (b.dtype != torch.float32 or not b.is_contiguous()):
            b = b.float().contiguous()
        code = DTYPE_CODE[x.dtype]
        call("clt_fp8_pass_fwd", crosslayer, x, code, ld, z, W, blocks, DTYPE_CODE[w_dtype], b, y, x_copy, w_copy, scratch, n, B, L, K,
             N, status, stream_ptr())
    return y, x_copy, w_copy


def _pass_backward(crosslayer, g, x_copy, w_copy, K, x_dtype, w_dtype, need_x, need_w, need_b):
    """(dx [B, L, K], dW [L or pairs, K, N], db [L, N]), None for what is not needed."""
    status, dev = _status_word(), g.device
    B, L, N = g.shape
    new = torch.empty if B else torch.zeros
    dx = new(B, L, K, dtype=x_dtype, device=dev) if need_x else None
    dW = new(_pairs(L) if crosslayer else L, K, N, dtype=w_dtype, device=dev) if need_w else None
    db = new(L, N, dtype=torch.float32, device=dev) if need_b else None
    if B:
        n = lib().query("clt_fp8_pass_units", crosslayer, 1, need_x, need_w, need_b, B, L, K, N)
        scratch = torch.empty(256 * n, device=dev, **_BYTES)
        g, ld, z = _rows_first(g)
        lib().call("clt_fp8_pass_bwd", crosslayer, g, DTYPE_CODE[g.dtype], ld, z, x_copy, w_copy, dx, dW, DTYPE_CODE[w_dtype], db,
                   scratch, n, B, L, K, N, status, stream_ptr())
    return dx, dW, db


def _pairs(t: int) -> int:
    return t * (t + 1) // 2


class _Project(torch.autograd.Function):
    """(Shapes are brought into the form [B, L, D] in here: views made outside would be nodes of the graph.)"""

    @staticmethod
    def forward(ctx, x, W, b):
        need_x, need_w = ctx.needs_input_grad[:2]
        ctx.shapes = xs, ws, _ = x.shape, W.shape, None if b is None else b.shape
        ctx.types = x.dtype, W.dtype, None if b is None else b.dtype
        L, (K, N) = 1 if len(ws) == 2 else ws[0], ws[-2:]
        if len(ws) == 2 or len(xs) != 3:
            x = x.reshape(xs.numel() // (L * K), L, K)
        if not W.is_contiguous():
            W = W.contiguous()
        y, x_copy, w_copy = _on(x.device, _pass_forward, 0, x, W, None, W.dtype, b, (*xs[:-1], N))
        ctx.dims = x.shape[0], L, K, N
        ctx.save_for_backward(x_copy if need_w else None, w_copy if need_x else None)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, g):
        B, L, K, N = ctx.dims
        xs, ws, bs = ctx.shapes
        x_copy, w_copy = ctx.saved_tensors
        dx, dW, db = _on(g.device, _pass_backward, 0, g.reshape(B, L, N), x_copy, w_copy, K, ctx.types[0], ctx.types[1],
                         *ctx.needs_input_grad)
        if db is not None and ctx.types[2] != torch.float32:
            db = db.to(ctx.types[2])
        if len(xs) == 3 and len(ws) == 3:
            return dx, dW, db
        return (None if dx is None else dx.view(xs), None if dW is None else dW.view(ws), None if db is None else db.view(bs))


def project(x: torch.Tensor, W: torch.Tensor, b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., L, D] -> [..., L, F]`` by layer ``l``'s ``W[l] [D, F]`` (and ``b [L, F]``), as ``Encoder.forward`` and the
    per-layer ``Decoder.forward``; or ``x [..., D]`` by one ``W [D, F]`` (and ``b [F]``).  Operands in 8 bits, result in ``x``'s type.
    Differentiable in ``x``, ``W`` and ``b``: backward reads the 8-bit copies of ``x`` and ``W`` that forward made and quantises
    the incoming gradient; one call keeps ``B L D + L D F`` bytes."""
    _check("x", x, DTYPE_CODE)
    _check("W", W, DTYPE_CODE, x.device)
    ws, xs = W.shape, x.shape
    one = len(ws) == 2
    if not one and len(ws) == 3 and ws[0] > 361:
        raise ValueError(f"{ws[0]} layers: at most 361 are supported")
    if len(ws) not in (2, 3) or W.numel() == 0:
        raise ValueError(f"expected W [D, F] or [L, D, F], not empty, got {tuple(ws)}")
    inner = 1 if one else 2
    if len(xs) < inner or xs[len(xs) - inner:] != ws[:inner]:
        raise ValueError(f"x {tuple(xs)} does not match W {tuple(ws)}")
    if b is not None:
        _check("b", b, DTYPE_CODE, x.device)
        if b.shape != (ws[-1:] if one else (ws[0], ws[2])):
            raise ValueError(f"b {tuple(b.shape)} does not match W {tuple(ws)}")
    _fits("x", xs.numel() // ws[:inner].numel(), ws[-2])
    _fits("W", ws[-2], ws[-1])
    return _Project.apply(x, W, b)


class _CrosslayerDecode(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, b, *blocks):
        need_w = any(ctx.needs_input_grad[2:])
        shape = ctx.shape = f.shape
        ctx.types = f.dtype, None if b is None else b.dtype, [w.dtype for w in blocks]
        (L, F), D = shape[-2:], blocks[0].shape[2]
        if len(shape) != 3:
            f = f.reshape(shape.numel() // (L * F), L, F)
        dtype = blocks[0].dtype
        if not all(w.dtype == dtype and w.is_contiguous() for w in blocks):
            dtype = torch.float32
            blocks = [w.float().contiguous() for w in blocks]
        at = array("Q", [w.data_ptr() for w in blocks])
        y, f_copy, w_copy = _on(f.device, _pass_forward, 1, f, None, at.buffer_info()[0], dtype, b, (*shape[:-1], D))
        ctx.dims = f.shape[0], L, F, D
        ctx.save_for_backward(f_copy if need_w else None, w_copy if ctx.needs_input_grad[0] else None)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, g):
        B, L, F, D = ctx.dims
        need_f, need_b, *need_w = ctx.needs_input_grad
        f_copy, w_copy = ctx.saved_tensors
        f_type, b_type, w_types = ctx.types
        same = w_types[0] if all(t == w_types[0] for t in w_types) else torch.float32
        df, dW, db = _on(g.device, _pass_backward, 1, g.reshape(B, L, D), f_copy, w_copy, F, f_type, same, need_f, any(need_w), need_b)
        if db is not None and b_type != torch.float32:
            db = db.to(b_type)
        parts = [None] * L
        if dW is not None:
            parts = [(p if dt == same else p.to(dt)) if need else None
                     for p, dt, need in zip(dW.split(list(range(1, L + 1))), w_types, need_w)]
        return (None if df is None else df.view(ctx.shape), db, *parts)


def crosslayer_decode(features: torch.Tensor, blocks: Sequence[torch.Tensor], b: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``features [..., L, F] -> [..., L, D]``: target layer ``t`` gets ``sum over s <= t of features[..., s, :] @ blocks[t][s]`` (and
    ``b[t]``), ``blocks[t]`` being ``[t + 1, F, D]``, as ``CrosslayerDecoder.forward``.  Types, rounding and what is kept for backward as
    in ``project``: ``B L F + P F D`` bytes for the P blocks of the decoder."""
    _check("features", features, DTYPE_CODE)
    shape, blocks = features.shape, list(blocks)
    if len(shape) < 2 or shape[-2] == 0 or len(blocks) != shape[-2]:
        raise ValueError(f"{len(blocks)} decoder blocks do not match features {tuple(shape)}")
    L, F = shape[-2:]
    if L > 361:
        raise ValueError(f"{L} layers: at most 361 are supported")
    for t, w in enumerate(blocks):
        _check(f"blocks[{t}]", w, DTYPE_CODE, features.device)
    D = blocks[0].shape[-1] if blocks[0].dim() else 0
    for t, w in enumerate(blocks):
        if w.shape != (t + 1, F, D) or F * D == 0:
            raise ValueError(f"blocks[{t}] {tuple(w.shape)} does not match {(t + 1, F, D)}, not empty")
    if b is not None:
        _check("b", b, DTYPE_CODE, features.device)
        if b.shape != (L, D):
            raise ValueError(f"b {tuple(b.shape)} does not match {(L, D)}")
    _fits("features", shape.numel() // (L * F), F)
    _fits("blocks", F, D)
    return _CrosslayerDecode.apply(features, b, *blocks)


def _jump_relu_forward(x, C, theta, bw, bw_value):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    R = y.numel() // C if C else 0
    ld = C
    if not x.is_contiguous():
        x = x.reshape(R, C)
        if x.stride(1) != 1 and C > 1:
            x = x.contiguous()
        ld = x.stride(0)
    bits = torch.empty(R, (C + 7) // 8, dtype=torch.int16, device=x.device)
    if R * C:
        lib().call("clt_jump_relu_fwd", x, ld, theta, bw, bw_value, y, bits, DTYPE_CODE[x.dtype], R, C, stream_ptr())
    return y, bits


def _jump_relu_backward(g, C, bits, theta, bw, bw_value):
    dx = torch.empty(g.shape, dtype=g.dtype, device=g.device)
    R = dx.numel() // C if C else 0
    ld = C
    if not g.is_contiguous():
        g = g.reshape(R, C)
        if g.stride(1) != 1 and C > 1:
            g = g.contiguous()
        ld = g.stride(0)
    if theta is None:
        dtheta, ws, n = None, None, 0
    else:
        dtheta = torch.empty(theta.shape, dtype=torch.float32, device=g.device)
        n = lib().query("clt_jump_relu_chunks", R, C) * C
        ws = torch.empty(n, dtype=torch.float32, device=g.device)
    if R * C:
        lib().call("clt_jump_relu_bwd", g, ld, bits, theta, bw, bw_value, dx, dtheta, ws, n, DTYPE_CODE[g.dtype], R, C,
                   stream_ptr())
    elif dtheta is not None:
        dtheta.zero_()
    return dx, dtheta


class _JumpReLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, theta, bandwidth, C):
        th, bw, value = theta, None, 0.0
        if theta is not None:
            if th.dtype != torch.float32 or not th.is_contiguous():
                th = th.float().contiguous()
            if isinstance(bandwidth, torch.Tensor):
                bw = bandwidth if bandwidth.dtype == torch.float32 else bandwidth.float()
            else:
                value = float(bandwidth)
        y, bits = _on(x.device, _jump_relu_forward, x, C, th, bw, value)
        ctx.value, ctx.C = value, C
        # (where the gradient passes, the bits say by themselves)
        ctx.save_for_backward(bits, *((theta, bw) if ctx.needs_input_grad[1] else (None, None)))
        return y

    @staticmethod
    @_first_order
    def backward(ctx, g):
        bits, theta, bw = ctx.saved_tensors
        th = theta
        if th is not None and (th.dtype != torch.float32 or not th.is_contiguous()):
            th = th.float().contiguous()
        dx, dtheta = _on(g.device, _jump_relu_backward, g, ctx.C, bits, th, bw, ctx.value)
        if dtheta is not None and theta.dtype != torch.float32:
            dtheta = dtheta.to(theta.dtype)
        return dx, dtheta, None, None


def jump_relu(x: torch.Tensor, theta: Optional[torch.Tensor] = None, bandwidth=1.0) -> torch.Tensor:
    """JumpReLU ``x [x > theta and x > 0]`` with the thresholds ``theta`` (``x``'s last axes, e.g. ``[L, F]`` or ``[1, L, F]``
    for ``x [..., L, F]``), or ReLU without.  Differentiable in ``x`` and ``theta`` as ``model.JumpReLU``: ``dx = g [x >= 0]`` (ReLU:
    ``[x > 0]``), ``dtheta = -(theta / bandwidth) sum g [theta - bandwidth / 2 < x <= theta + bandwidth / 2]``, from two bits an
    element instead of ``x``.  A masked element is 0 and gets no gradient whatever it was; NaN stays NaN.  ``bandwidth``: a positive number,
    or one on ``x``'s device."""
    _check("x", x, DTYPE_CODE)
    shape = x.shape
    if len(shape) == 0:
        raise ValueError("x has no axis")
    C = shape[-1]
    if theta is not None:
        _check("theta", theta, DTYPE_CODE, x.device)
        inner = theta.shape
        while len(inner) > 1 and inner[0] == 1 and inner != shape[len(shape) - len(inner):]:
            inner = inner[1:]
        if not 1 <= len(inner) <= len(shape) or inner != shape[len(shape) - len(inner):]:
            raise ValueError(f"theta {tuple(theta.shape)} does not match the last axes of x {tuple(shape)}")
        C = inner.numel()
        if isinstance(bandwidth, torch.Tensor):
            _check("bandwidth", bandwidth, DTYPE_CODE, x.device)
            if bandwidth.numel() != 1:
                raise ValueError(f"bandwidth has {bandwidth.numel()} elements")
        elif not float(bandwidth) > 0:
            raise ValueError(f"bandwidth must be positive, got {bandwidth}")
    _fits("x", x.numel() // C if C else 0, C)
    return _JumpReLU.apply(x, theta, bandwidth, C)
