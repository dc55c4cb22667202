"""The 8-bit operators as they are used together: in the model, on streams, in graphs, on large tensors."""
import threading

import pytest
import torch

from crosslayer_transcoder_b200 import fp8
from crosslayer_transcoder_b200.model import (CrossLayerTranscoder, CrossLayerTranscoderModule, CrosslayerDecoder, Decoder,
                                              DimensionwiseInputStandardizer, DimensionwiseOutputStandardizer, Encoder,
                                              JumpReLU, PerLayerTopK, ReLU)
from tests import fp8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _model(L, D, F, nl, crosslayer, seed=0):
    torch.manual_seed(seed)
    dec = (CrosslayerDecoder if crosslayer else Decoder)(D, F, L)
    model = CrossLayerTranscoder(nl, Encoder(D, F, L), dec, DimensionwiseInputStandardizer(L, D), DimensionwiseOutputStandardizer(L, D))
    with torch.no_grad():
        model.encoder.b.normal_(0, 0.1)
        dec.b.normal_(0, 0.1)
    model = model.to(DEV)
    model.initialize_standardizers(torch.randn(64, 2, L, D, device=DEV))
    return model


KINDS = [("jumprelu", True), ("jumprelu", False), ("relu", True), ("topk", False)]


@pytest.mark.parametrize("kind, crosslayer", KINDS)
def test_model_forward_and_backward(kind, crosslayer):
    """The switched model is the operators one after another, and near the eager model: a product's rounding is at most
    (1 + 2^-4)^2 - 1 of the magnitudes it sums, and what a block flushes, 2^-18 of its largest element by the other operand."""
    L, D, F, B = 3, 96, 200, 150
    nl = {"jumprelu": lambda: JumpReLU(0.03, 1.0, L, F), "relu": ReLU, "topk": lambda: PerLayerTopK(k=16)}[kind]()
    model = _model(L, D, F, nl, crosslayer)
    x = torch.randn(B, L, D, device=DEV, requires_grad=True)
    eager = model(x)
    model.eight_bit = True
    out = model(x)
    params = list(model.parameters())
    g = torch.randn_like(out[3])
    grads = torch.autograd.grad(out[3], [x, *params], g)
    xs = model.input_standardizer(x)
    pre = fp8.project(xs, model.encoder.W, model.encoder.b)
    feats = fp8.jump_relu(pre, nl.theta, nl.bandwidth) if kind == "jumprelu" else torch.relu(pre) if kind == "relu" else nl(pre)
    rec = fp8.crosslayer_decode(feats, model.decoder.blocks(), model.decoder.b) if crosslayer else \
        fp8.project(feats, model.decoder.W, model.decoder.b)
    full = model.output_standardizer(rec)
    want = torch.autograd.grad(full, [x, *params], g)
    assert all(torch.equal(a, b) for a, b in zip(out, (pre, feats, rec, full)))
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    W = model.encoder.W
    mags = torch.einsum("bld,ldf->blf", xs.abs(), W.abs())
    flush = 2.0 ** -18 * D * xs.abs().max() * W.abs().max() * 2
    assert bool(((pre - eager[0]).abs() <= ((1 + 2.0 ** -4) ** 2 - 1) * mags + flush + 1e-5).all())
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(model(x), out))
    fp8.check_status()


def test_module_forward_uses_the_switch():
    model = _model(2, 64, 256, JumpReLU(0.03, 1.0, 2, 256), True)
    module = CrossLayerTranscoderModule(model=model)
    x = torch.randn(40, 2, 64, device=DEV)
    with torch.no_grad():
        infer = module(x)
        model.eight_bit = True
        switched = module(x)
        assert all(torch.equal(a, b) for a, b in zip(switched, model(x)))
    assert not torch.equal(switched[0], infer[0])


def test_training_steps_through_the_switched_model():
    """Steps of a plain optimizer on the differentiable forward: every parameter gets a finite gradient and moves."""
    model = _model(3, 64, 300, JumpReLU(0.03, 1.0, 3, 300), True)
    model.eight_bit = True
    opt = torch.optim.SGD(model.parameters(), lr=1e-3)
    x, y = torch.randn(100, 3, 64, device=DEV), torch.randn(100, 3, 64, device=DEV)
    before = [p.detach().clone() for p in model.parameters()]
    for _ in range(3):
        opt.zero_grad()
        ((model(x)[2] - y) ** 2).sum().backward()
        assert all(torch.isfinite(p.grad).all() and p.grad.any() for p in model.parameters())
        opt.step()
    assert all(not torch.equal(p, b) for p, b in zip(model.parameters(), before))


def test_what_a_pass_keeps():
    """Bytes that autograd holds between forward and backward: one per input, feature and decoder weight, two bits per
    pre-activation; none for the encoder's weights, which only the input's gradient would read, and the input needs none."""
    L, D, F, B = 4, 128, 1024, 512
    model = _model(L, D, F, JumpReLU(0.03, 1.0, L, F), True)
    model.input_standardizer = model.output_standardizer = None
    x = torch.randn(B, L, D, device=DEV)

    def kept(eight_bit):
        model.eight_bit = eight_bit
        seen = {}
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.setdefault((t.data_ptr(), t.numel()), t) if t.is_cuda else t, lambda t: t):
            model(x)
        params = {p.data_ptr() for p in model.parameters()}
        return sum(t.numel() * t.element_size() for (p, _), t in seen.items() if p not in params)

    P = L * (L + 1) // 2
    values = B * L * D + B * L * F + P * F * D + B * L * F // 4
    assert values <= kept(True) <= 1.01 * values


# ---- streams and graphs ----------------------------------------------------------------------------------------------------------
def _leaves(seed, B=140, L=2, D=96, F=200):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, L, D, device=DEV, generator=g, requires_grad=True)
    W = (torch.randn(L, D, F, device=DEV, generator=g) * 0.1).requires_grad_()
    ws = [(torch.randn(t + 1, F, D, device=DEV, generator=g) * 0.1).requires_grad_() for t in range(L)]
    th = (torch.rand(L, F, device=DEV, generator=g) * 0.1).requires_grad_()
    return x, W, th, ws


def _pass(x, W, th, ws):
    y = fp8.crosslayer_decode(fp8.jump_relu(fp8.project(x, W), th, 1.0), ws)
    return (y.detach(), *torch.autograd.grad(y, (x, W, th, *ws), torch.ones_like(y)))


def test_two_streams_and_threads_at_once():
    leaves = [_leaves(s) for s in range(4)]
    want = [_pass(*l) for l in leaves]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream(DEV)):
            for _ in range(20):
                got[i] = _pass(*leaves[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    fp8.check_status()


def test_captured_and_replayed():
    """Two graphs with passes of their own, replayed with new inputs in turn and one after another without waiting."""
    _pass(*_leaves(0))                                      # (kernels are loaded, the status word exists)
    torch.cuda.synchronize()
    made = []
    for s in range(2):
        leaves = _leaves(s)
        stream = torch.cuda.Stream(DEV)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _pass(*leaves)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _pass(*leaves)
        made.append((graph, leaves, out))
    for s in (5, 6):
        fresh = _leaves(s)
        want = _pass(*fresh)
        for graph, leaves, _ in made:
            with torch.no_grad():
                for dst, src in zip((*leaves[:3], *leaves[3]), (*fresh[:3], *fresh[3])):
                    dst.copy_(src)
            graph.replay()
        for _, _, out in made:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    fp8.check_status()


def test_captured_product_of_parts():
    """A product that is cut into parts has scratch of its own in every graph."""
    a = fp8.quantize(torch.randn(20, 9000, device=DEV), 1)
    b = fp8.quantize(torch.randn(9000, 130, device=DEV))
    want = fp8.matmul(a, b, out_dtype=torch.float32)
    outs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8.matmul(a, b, out_dtype=torch.float32)
        outs.append((graph, y))
    s = [torch.cuda.Stream(DEV) for _ in outs]
    for _ in range(10):
        for st, (graph, y) in zip(s, outs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for _, y in outs)


def test_kernel_that_a_capture_meets_first():
    """Another type and layout than any call before: what its kernel needs is set up inside the capture."""
    a, b = fp8.quantize(torch.randn(300, 200, device=DEV)), fp8.quantize(torch.randn(200, 136, device=DEV))
    fp8.matmul(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.matmul(b.mT, a.mT, out_dtype=torch.float16)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, fp8.matmul(b.mT, a.mT, out_dtype=torch.float16))


def test_first_call_in_a_capture_is_refused(monkeypatch):
    """Nothing is allocated for the status word while a graph is being captured."""
    monkeypatch.setattr(fp8, "_status", None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(fp8.CltError, match="before a graph is captured"):
        fp8.matmul(fp8.quantize(torch.zeros(4, 4, device=DEV)), fp8.quantize(torch.zeros(4, 4, device=DEV)))


def test_backward_twice_is_refused():
    """A second derivative is not offered, and a retained graph gives the same gradients again."""
    x, W, _, _ = _leaves(1)
    y = fp8.project(x, W)
    a = torch.autograd.grad(y, (x, W), torch.ones_like(y), retain_graph=True)
    b = torch.autograd.grad(y, (x, W), torch.ones_like(y))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    y = fp8.project(x, W)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_weights_changed_between_forward_and_backward():
    """Backward goes by the operands of its forward."""
    x, W, _, _ = _leaves(2)
    y = fp8.project(x, W)
    want = torch.autograd.grad(y, (x, W), torch.ones_like(y), retain_graph=True)
    with torch.no_grad():
        W.mul_(3.0)
        x.add_(1.0)
    got = torch.autograd.grad(y, (x, W), torch.ones_like(y))
    assert all(torch.equal(u, v) for u, v in zip(got, want))


# ---- large tensors ---------------------------------------------------------------------------------------------------------------
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in an operand, a result and a checkpoint; the last rows against the same rows alone."""
    R, C = 70001, 32768
    x = torch.zeros(R, C, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(129, C, device=DEV).bfloat16()
    x[-129:] = tail
    pad = R % 128                                           # the last block of rows has R % 128 of them
    for rows in (1, 128):
        q = fp8.quantize(x, rows)
        alone = fp8.quantize(tail[-pad:].contiguous(), rows)
        assert torch.equal(q.values[-pad:].float(), alone.values.float())
        assert torch.equal(q.scales[-alone.scales.shape[0]:], alone.scales)
        back = q.dequantize(torch.bfloat16)
        assert torch.equal(back[-pad:], alone.dequantize(torch.bfloat16)) and not back[:R - 300].any()
        del back
        w = fp8.quantize(torch.randn(C, 128, device=DEV))
        y = fp8.matmul(q, w)
        # (the rows alone are cut into parts along C, which are other bits)
        va, vw = alone.dequantize().double().cpu(), w.dequantize().double().cpu()
        ref.check(y[-pad:], va @ vw, va.abs() @ vw.abs(), C)
        assert not y[:R - 300].any()
    del q, y
    a = fp8.quantize(torch.randn(R, 128, device=DEV), 1)
    w = fp8.quantize(torch.randn(128, C, device=DEV))
    y = fp8.matmul(a, w)
    last = fp8.BlockTensor(a.values[-200:], a.scales[-200:], 1)
    assert torch.equal(y[-200:], fp8.matmul(last, w))
    del y
    th = torch.full((C,), 0.03, device=DEV)
    xr = x.requires_grad_()
    f = fp8.jump_relu(xr, th)
    g = torch.zeros_like(x)
    g[-129:] = 1
    (dx,) = torch.autograd.grad(f, xr, g)
    small = tail.clone().requires_grad_()
    fs = fp8.jump_relu(small, th)
    assert torch.equal(f[-129:], fs) and torch.equal(dx[-129:], torch.autograd.grad(fs, small, torch.ones_like(fs))[0])
    fp8.check_status()
