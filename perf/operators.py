"""What the speed of the 8-bit operators (``crosslayer_transcoder_b200.fp8``) is measured on.

Five operators:

``quantize``  activations in 8 bits and back: e4m3 values with a power-of-two scale for each block of 1 x 128 or 128 x 128.
``matmul``    product of two such operands, with a bias, in fp32 sums.
``project``   a training pass through an encoder or a per-layer decoder whose operands are in 8 bits, the input among them:
              that copy is what backward reads.
``decode``    the same for the crosslayer decoder (every source layer writes to every later target layer).
``jumprelu``  (Jump)ReLU whose checkpoint is two bits an element: forward and backward.

A scale is the smallest power of two that brings its block's largest magnitude to at most 448, the largest e4m3 value.
"""
import math

import torch

#: The tools set it: the framework's operators (true) or their plain form (false).
own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_THETA, _BANDWIDTH = 0.03, 1.0


def _quantize_case(name, Z, R, C, rows, dtype):
    return _named(name, {"op": "quantize", "Z": Z, "R": R, "C": C, "rows": rows, "dtype": dtype})


def _matmul_case(name, G, M, K, N, rows, a_t, b_t, bias, out):
    return _named(name, {"op": "matmul", "G": G, "M": M, "K": K, "N": N, "rows": rows, "a_t": a_t, "b_t": b_t,
                         "bias": bias, "out": out})


def _layers_case(op, name, B, L, D, F, dtype):
    return _named(name, {"op": op, "B": B, "L": L, "D": D, "F": F, "dtype": dtype})


def _jumprelu_case(name, B, L, F, dtype, theta):
    return _named(name, {"op": "jumprelu", "B": B, "L": L, "F": F, "dtype": dtype, "theta": theta})


def _named(name, case):
    return dict(case, name=name) if name else case


def listed():
    return [
        # The test-suite's width: launches and latency.
        _quantize_case("quantize tiny", 3, 136, 64, 128, "fp32"),
        # The encoder's input of the benchmark batch, rows scaled one by one for an inference product.
        _quantize_case("quantize inputs", 12, 4000, 768, 1, "bf16"),
        # The features of the reference's default training configuration, kept from forward to backward: no block
        # divides the 10000 columns or the 4000 tokens.
        _quantize_case("quantize features", 12, 4000, 10000, 128, "bf16"),
        # One token through one layer's encoder of the per-layer transcoder: the weights are all there is to read.
        _matmul_case("matmul one token", 1, 1, 768, 24576, 1, False, False, True, "bf16"),
        # One prompt's tokens through the last target of the default crosslayer decoder: the features of all twelve layers
        # in one long contraction, few output tiles.
        _matmul_case("matmul decode prompt", 1, 257, 120000, 768, 1, False, False, True, "fp32"),
        # All layers' pre-activations of a benchmark batch.
        _matmul_case("matmul encode batch", 12, 4000, 768, 24576, 1, False, False, True, "bf16"),
        # Debugging run at the test-suite's size.
        _layers_case("project", "project tiny", 136, 3, 64, 256, "fp32"),
        # Encoder of the per-layer transcoder of the benchmark set, one training pass.
        _layers_case("project", "project encoder", 4000, 12, 768, 24576, "bf16"),
        # Ragged batch through a small crosslayer decoder with a feature count that no block divides.
        _layers_case("decode", "decode odd", 777, 6, 320, 2001, "fp32"),
        # The reference's default crosslayer decoder, one training pass.
        _layers_case("decode", "decode default", 4000, 12, 768, 10000, "bf16"),
        # Pre-activations of the reference's CPU-runnable toy configuration, in full precision.
        _jumprelu_case("jumprelu toy", 512, 12, 1024, "fp32", True),
        # Pre-activations of the per-layer transcoder of the benchmark set.
        _jumprelu_case("jumprelu features", 4000, 12, 24576, "bf16", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(["quantize", "matmul", "matmul", "project", "project", "decode", "jumprelu"])
        dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
        if op == "quantize":
            c = _quantize_case(None, rng.randint(1, 12), _log(rng, 1, 8192), _log(rng, 16, 32768), rng.choice([1, 128]), dtype)
        elif op == "matmul":
            rows = rng.choice([1, 128])
            c = _matmul_case(None, rng.randint(1, 12), _log(rng, 1, 8192), _log(rng, 64, 120000), _log(rng, 64, 32768), rows,
                             rows == 128 and rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5,
                             rng.choice(["bf16", "fp32", "fp16"]))
        elif op == "project":
            c = _layers_case(op, None, _log(rng, 64, 8192), rng.randint(1, 12), _log(rng, 64, 2304), _log(rng, 200, 32768), dtype)
        elif op == "decode":
            c = _layers_case(op, None, _log(rng, 64, 6000), rng.randint(2, 12), _log(rng, 64, 2304), _log(rng, 200, 16384), dtype)
        else:
            c = _jumprelu_case(None, _log(rng, 64, 8192), rng.randint(1, 16), _log(rng, 200, 32768), dtype, rng.random() < 0.7)
        w = work(c)
        if op == "matmul" and max(c["G"] * c["M"] * c["K"], c["G"] * c["K"] * c["N"], c["G"] * c["M"] * c["N"]) > 10 ** 9:
            continue        # the plain form holds its operands in 32 bits
        # none costs more than the largest listed one, and three states with their outputs fit the card
        if w["flops"] <= max(m["flops"] for m in most) and w["bytes"] <= min(1.2e10, max(m["bytes"] for m in most)):
            return c


def _blocks(n):
    return -(-n // 128)


def _pairs(L):
    return L * (L + 1) // 2


def work(case):
    c, op = case, case["op"]
    if op == "quantize":
        n, e = float(c["Z"] * c["R"] * c["C"]), _BYTES[c["dtype"]]
        scales = 4.0 * c["Z"] * -(-c["R"] // c["rows"]) * _blocks(c["C"])
        # written in 8 bits, and read again for the copy that comes back
        return {"bytes": n * (e + 1 + 1 + e) + 2 * scales, "flops": 2 * n}
    if op == "matmul":
        G, M, K, N = (float(c[k]) for k in "GMKN")
        return {"bytes": G * (M * K + K * N + M * N * _BYTES[c["out"]]), "flops": 2 * G * M * K * N}
    B, L, F = float(c["B"]), c["L"], float(c["F"])
    e = _BYTES[c["dtype"]]
    if op == "jumprelu":
        n = B * L * F
        return {"bytes": 4 * e * n + 2 * n / 4 + 8 * L * F, "flops": 6 * n}
    D = float(c["D"])
    if op == "project":
        # x, W and dy come in, y, dx and dW go out; the 8-bit copies of x and W are written, and read in backward
        return {"bytes": 2 * e * B * L * (D + F) + 8 * L * D * F + 2 * (B * L * D + L * D * F), "flops": 6 * B * L * D * F}
    P = _pairs(L)
    return {"bytes": 2 * e * B * L * (D + F) + 8 * P * D * F + 2 * (B * L * F + P * D * F), "flops": 6 * B * P * D * F}


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _acts(shape, g, dev, dtype):
    """Activations: every dimension of the last axis has its own spread, a few of them twenty times as large."""
    spread = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=dev))
    spread[torch.randint(shape[-1], (max(1, shape[-1] // 192),), generator=g, device=dev)] *= 20.0
    return (torch.randn(shape, generator=g, device=dev) * spread).to(dtype)


def _features(shape, g, dev, dtype):
    """Features: one in six above its threshold, none below zero."""
    return torch.relu(torch.randn(shape, generator=g, device=dev) - 1.0).to(dtype)


def _weights(shape, g, dev, bound):
    return torch.empty(shape, device=dev).uniform_(-bound, bound, generator=g)


def prepare(case, seed):
    c, dev = case, torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    op, s = c["op"], {"case": c}
    if op == "quantize":
        make = _features if c["C"] > 4096 else _acts
        s["x"] = make((c["Z"], c["R"], c["C"]), g, dev, _TYPES[c["dtype"]])
    elif op == "matmul":
        G, M, K, N = (c[k] for k in "GMKN")
        s["a"] = _quantize(_acts((G, K, M) if c["a_t"] else (G, M, K), g, dev, torch.float32), c["rows"])
        s["b"] = _quantize(_weights((G, N, K) if c["b_t"] else (G, K, N), g, dev, K ** -0.5), 128)
        s["bias"] = 0.1 * torch.randn(G, N, generator=g, device=dev) if c["bias"] else None
    elif op == "jumprelu":
        B, L, F, t = c["B"], c["L"], c["F"], _TYPES[c["dtype"]]
        s["pre"] = (0.5 * torch.randn(B, L, F, generator=g, device=dev)).to(t).requires_grad_()
        s["theta"] = None
        if c["theta"]:
            s["theta"] = (_THETA * (0.5 + torch.rand(L, F, generator=g, device=dev))).requires_grad_()
        s["grad"] = (1e-3 * torch.randn(B, L, F, generator=g, device=dev)).to(t)
    else:
        B, L, D, F, t = c["B"], c["L"], c["D"], c["F"], _TYPES[c["dtype"]]
        if op == "project":
            s["x"] = _acts((B, L, D), g, dev, t).requires_grad_()
            s["W"] = _weights((L, D, F), g, dev, D ** -0.5).requires_grad_()
            s["b"] = (0.02 * torch.randn(L, F, generator=g, device=dev)).requires_grad_()
            s["grad"] = (1e-3 * torch.randn(B, L, F, generator=g, device=dev)).to(t)
        else:
            s["x"] = _features((B, L, F), g, dev, t).requires_grad_()
            s["W"] = [_weights((i + 1, F, D), g, dev, (L * F) ** -0.5).requires_grad_() for i in range(L)]
            s["b"] = (0.02 * torch.randn(L, D, generator=g, device=dev)).requires_grad_()
            s["grad"] = (1e-3 * torch.randn(B, L, D, generator=g, device=dev)).to(t)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------


def _quantize(x, rows):
    """(values in e4m3 [Z, R, C], scales [Z, R / rows, C / 128]) of x [Z, R, C]."""
    Z, R, C = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -C % 128, 0, -R % rows))
    x = x.view(Z, x.shape[1] // rows, rows, x.shape[2] // 128, 128)
    amax = x.abs().amax(dim=(2, 4))
    # amax = m 2^e with m in [1/2, 1), and 448 = 0.875 * 2^9
    m, e = torch.frexp(amax)
    e = torch.clamp(torch.where(m <= 0.875, e - 9, e - 8), min=-126)
    scale = ((e + 127).to(torch.int32) << 23).view(torch.float32)
    scale = torch.where(amax == 0, torch.ones_like(scale), scale)
    values = (x / scale[:, :, None, :, None]).to(torch.float8_e4m3fn)
    values = values.view(Z, x.shape[1] * rows, x.shape[3] * 128)[:, :R, :C]
    return values.contiguous(), scale


def _dequantize(q, rows):
    values, scale = q
    R, C = values.shape[-2:]
    s = scale.repeat_interleave(rows, dim=-2)[..., :R, :].repeat_interleave(128, dim=-1)[..., :C]
    return values.float() * s


def _rounded(x, rows=128):
    """x [Z, R, C] as its 8-bit form stands for it."""
    return _dequantize(_quantize(x, rows), rows)


def _plain_project(s):
    x, W, b, g = s["x"].detach(), s["W"].detach(), s["b"].detach(), s["grad"]
    xq, Wq, gq = _rounded(x.transpose(0, 1)), _rounded(W), _rounded(g.transpose(0, 1))
    y = torch.matmul(xq, Wq) + b[:, None]
    dx = torch.matmul(gq, Wq.transpose(1, 2))
    return {"y": y.transpose(0, 1).to(x.dtype), "dx": dx.transpose(0, 1).to(x.dtype), "dW": torch.matmul(xq.transpose(1, 2), gq),
            "db": g.float().sum(dim=0)}


def _plain_decode(s):
    f, W, b, g = s["x"].detach(), [w.detach() for w in s["W"]], s["b"].detach(), s["grad"]
    L = f.shape[1]
    fq, gq, Wq = _rounded(f.transpose(0, 1)), _rounded(g.transpose(0, 1)), [_rounded(w) for w in W]
    y = [torch.matmul(fq[:t + 1], Wq[t]).sum(dim=0) + b[t] for t in range(L)]
    dx = [sum(torch.matmul(gq[t], Wq[t][i].t()) for t in range(i, L)) for i in range(L)]
    dW = [torch.matmul(fq[:t + 1].transpose(1, 2), gq[t]) for t in range(L)]
    return {"y": torch.stack(y, dim=1).to(f.dtype), "dx": torch.stack(dx, dim=1).to(f.dtype), "dW": dW,
            "db": g.float().sum(dim=0)}


def _plain_jumprelu(s):
    pre, g = s["pre"].detach(), s["grad"]
    x, zero = pre.float(), torch.zeros((), device=pre.device)
    if s["theta"] is None:
        return {"y": torch.where(x > 0, x, zero).to(pre.dtype), "dx": torch.where(x > 0, g, zero.to(g.dtype))}
    theta = s["theta"].detach()
    y = torch.where((x > theta) & (x > 0), x, zero).to(pre.dtype)
    u = (x.double() - theta.double()) / _BANDWIDTH
    inside = (u > -0.5) & (u <= 0.5)
    dtheta = -(theta / _BANDWIDTH) * torch.where(inside, g.float(), zero).sum(dim=0)
    return {"y": y, "dx": torch.where(x >= 0, g, zero.to(g.dtype)), "dtheta": dtheta}


# ---- one pass ---------------------------------------------------------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        return _own(s, c, op)
    if op == "quantize":
        q = _quantize(s["x"], c["rows"])
        return {"scales": q[1], "back": _dequantize(q, c["rows"]).to(s["x"].dtype)}
    if op == "matmul":
        a, b = _dequantize(s["a"], c["rows"]), _dequantize(s["b"], 128)
        y = torch.matmul(a.transpose(1, 2) if c["a_t"] else a, b.transpose(1, 2) if c["b_t"] else b)
        return (y if s["bias"] is None else y + s["bias"][:, None]).to(_TYPES[c["out"]])
    return {"project": _plain_project, "decode": _plain_decode, "jumprelu": _plain_jumprelu}[op](s)


def _own(s, c, op):
    from crosslayer_transcoder_b200 import fp8

    if op == "quantize":
        q = fp8.quantize(s["x"], block_rows=c["rows"])
        return {"scales": q.scales, "back": q.dequantize(s["x"].dtype)}
    if op == "matmul":
        a, b = fp8.BlockTensor(*s["a"], block_rows=c["rows"]), fp8.BlockTensor(*s["b"])
        return fp8.matmul(a.mT if c["a_t"] else a, b.mT if c["b_t"] else b, bias=s["bias"], out_dtype=_TYPES[c["out"]])
    if op == "jumprelu":
        y = fp8.jump_relu(s["pre"], s["theta"], _BANDWIDTH)
        if s["theta"] is None:
            return {"y": y.detach(), "dx": torch.autograd.grad(y, s["pre"], s["grad"])[0]}
        dx, dtheta = torch.autograd.grad(y, (s["pre"], s["theta"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dtheta": dtheta}
    if op == "project":
        y = fp8.project(s["x"], s["W"], s["b"])
        dx, dW, db = torch.autograd.grad(y, (s["x"], s["W"], s["b"]), s["grad"])
        return {"y": y.detach(), "dx": dx, "dW": dW, "db": db}
    y = fp8.crosslayer_decode(s["x"], s["W"], s["b"])
    dx, db, *dW = torch.autograd.grad(y, (s["x"], s["b"], *s["W"]), s["grad"])
    return {"y": y.detach(), "dx": dx, "dW": dW, "db": db}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------


def _exact8(x, rows):
    """(scale, value) in 64 bits of one matrix [R, C], from the format's definition: a scale is 2^ceil(log2(amax / 448)), and
    an e4m3 number has three bits behind its leading one, the smallest leading one being 2^-6."""
    x = x.detach().double()
    R, C = x.shape
    pad = torch.zeros(-(-R // rows) * rows, _blocks(C) * 128, dtype=torch.float64, device=x.device)
    pad[:R, :C] = x
    top = pad.unfold(0, rows, rows).unfold(1, 128, 128).abs().flatten(2).max(dim=2).values
    lead, power = torch.frexp(top / 448.0)          # lead 2^power with lead in [1/2, 1): a power of two has 1/2
    scale = torch.exp2((power - (lead == 0.5).to(power.dtype)).double().clamp(min=-126.0))
    scale[top == 0] = 1.0
    wide = torch.kron(scale, torch.ones(rows, 128, dtype=torch.float64, device=x.device))[:R, :C]
    v = x / wide
    step = torch.exp2((torch.frexp(v)[1] - 1).double().clamp(min=-6.0) - 3.0)
    return scale, torch.round(v / step) * step * wide


def _exact_values(q, rows):
    values, scale = q
    R, C = values.shape[1:]
    one = torch.ones(rows, 128, dtype=torch.float64, device=values.device)
    return torch.stack([v.double() * torch.kron(s.double(), one)[:R, :C] for v, s in zip(values, scale)])


def exact(case, seed):
    c, op = case, case["op"]
    s = prepare(case, seed)
    if op == "quantize":
        each = [_exact8(x, c["rows"]) for x in s["x"]]
        return {"scales": torch.stack([e[0] for e in each]), "back": torch.stack([e[1] for e in each])}
    if op == "matmul":
        a, b = _exact_values(s["a"], c["rows"]), _exact_values(s["b"], 128)
        y = torch.einsum(("gkm," if c["a_t"] else "gmk,") + ("gnk->gmn" if c["b_t"] else "gkn->gmn"), a, b)
        return y if s["bias"] is None else y.add_(s["bias"].double()[:, None, :])
    if op == "jumprelu":
        x, g = s["pre"].detach().double(), s["grad"].double()
        if s["theta"] is None:
            return {"y": x.clamp(min=0.0), "dx": g * (x > 0)}
        th = s["theta"].detach().double()
        near = (x > th - 0.5 * _BANDWIDTH) & ~(x > th + 0.5 * _BANDWIDTH)
        return {"y": x * ((x > th) & (x > 0)), "dx": g * ~(x < 0), "dtheta": (g * near).sum(dim=0) * -(th / _BANDWIDTH)}
    x, g, b = s["x"].detach(), s["grad"], s["b"].detach().double()
    L = c["L"]
    y, dx, dW = [], [], []
    if op == "project":
        for l in range(L):
            xl, wl, gl = _exact8(x[:, l], 128)[1], _exact8(s["W"][l], 128)[1], _exact8(g[:, l], 128)[1]
            y.append(torch.addmm(b[l], xl, wl))
            dx.append(gl @ wl.T)
            dW.append(xl.T @ gl)
        dW = torch.stack(dW)
    else:
        fl, gl = [_exact8(x[:, l], 128)[1] for l in range(L)], [_exact8(g[:, l], 128)[1] for l in range(L)]
        dx = [torch.zeros_like(f) for f in fl]
        for t in range(L):
            out, grads = b[t].expand(c["B"], -1).clone(), []
            for i in range(t + 1):
                w = _exact8(s["W"][t][i], 128)[1]
                out.addmm_(fl[i], w)
                dx[i].addmm_(gl[t], w.T)
                grads.append(fl[i].T @ gl[t])
            y.append(out)
            dW.append(torch.stack(grads))
    return {"y": torch.stack(y, dim=1), "dx": torch.stack(dx, dim=1), "dW": dW, "db": g.double().sum(dim=0)}
