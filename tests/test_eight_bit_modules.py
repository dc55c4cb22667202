"""What the 8-bit forward does with the modules of a transcoder, on the CPU: plain torch in place of the operators."""
import pytest
import torch
from torch import nn

from crosslayer_transcoder_b200.model import CrosslayerDecoder, CrossLayerTranscoder, Decoder, Encoder, JumpReLU, PerLayerTopK, ReLU
from tests import fp8_stand_in

L, D, F, B = 3, 8, 16, 6
NONLINEARITIES = [lambda: JumpReLU(0.03, 1.0, L, F), ReLU, nn.ReLU, lambda: PerLayerTopK(k=2)]


@pytest.fixture(autouse=True)
def _stand_in(monkeypatch):
    fp8_stand_in.install(monkeypatch.setattr)


def _model(nl, decoder=CrosslayerDecoder, encoder=Encoder):
    torch.manual_seed(2)
    return CrossLayerTranscoder(nl, encoder(D, F, L), decoder(D, F, L))


def _both(model, x):
    """(eager results, 8-bit ones)."""
    model.eight_bit = False
    eager = model(x)
    model.eight_bit = True
    return eager, model(x)


@pytest.mark.parametrize("decoder", [CrosslayerDecoder, Decoder])
@pytest.mark.parametrize("nl", NONLINEARITIES)
def test_hooks_run(nl, decoder):
    """Forward, pre- and backward hooks on encoder, nonlinearity and decoder run, once, and what they return is used."""
    model = _model(nl(), decoder)
    x = torch.randn(B, L, D)
    plain = _both(model, x)[1]
    seen = []
    for name in ("encoder", "nonlinearity", "decoder"):
        m = getattr(model, name)
        m.register_forward_pre_hook(lambda m, args, name=name: seen.append(("pre", name)))
        m.register_forward_hook(lambda m, args, out, name=name: seen.append(("post", name)))
        m.register_full_backward_hook(lambda m, gin, gout, name=name: seen.append(("back", name)))
    out = model(x)
    assert all(torch.equal(a, b) for a, b in zip(out, plain))
    out[2].sum().backward()
    order = ["encoder", "nonlinearity", "decoder"]
    assert seen == [(when, n) for n in order for when in ("pre", "post")] + [("back", n) for n in reversed(order)]
    handle = model.nonlinearity.register_forward_hook(lambda m, args, out: torch.zeros_like(out))    # an ablation
    assert torch.equal(model(x)[2], model.decoder.b.expand(B, L, D))
    handle.remove()
    model.encoder.register_forward_pre_hook(lambda m, args: (2 * args[0],))
    assert torch.equal(model(x)[0], _both(_model(nl(), decoder), 2 * x)[1][0])


def test_global_hooks_run():
    model, names = _model(nn.ReLU()), []
    model.eight_bit = True
    handle = nn.modules.module.register_module_forward_hook(lambda m, args, out: names.append(type(m).__name__))
    try:
        model(torch.randn(B, L, D))
    finally:
        handle.remove()
    assert names == ["Encoder", "ReLU", "CrosslayerDecoder", "CrossLayerTranscoder"]


class _Scaled(Encoder):
    def forward(self, acts_norm, layer="all"):
        return 3 * super().forward(acts_norm, layer)


class _Leaky(JumpReLU):
    def forward(self, input):
        return super().forward(input) + 0.1 * input


class _Leaky0(nn.ReLU):
    def forward(self, input):
        return super().forward(input) + 0.1 * input


class _Shifted(CrosslayerDecoder):
    def forward(self, features, layer="all"):
        return super().forward(features, layer) + 1


class _Decoder2(Decoder):
    def forward(self, features, layer="all"):
        return super().forward(features, layer) + 1


class _Kept(Encoder):
    """Another class with the same forward."""


@pytest.mark.parametrize("kw", [dict(encoder=_Scaled), dict(nl=_Leaky(0.03, 1.0, L, F)), dict(nl=_Leaky0()), dict(decoder=_Shifted),
                                dict(decoder=_Decoder2), dict(encoder=_Kept), dict(nl=nn.ReLU(inplace=True)), dict(nl=nn.GELU())])
def test_forwards_of_subclasses_are_kept(kw):
    model = _model(**{"nl": ReLU(), **kw})
    for a, b in zip(*_both(model, torch.randn(B, L, D))):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_forward_of_an_instance_is_kept():
    model = _model(ReLU())
    model.encoder.forward = lambda acts: torch.ones(B, L, F)
    model.eight_bit = True
    assert torch.equal(model(torch.randn(B, L, D))[0], torch.ones(B, L, F))


def test_own_forwards_reach_the_operators(monkeypatch):
    """With and without hooks; a subclass that keeps the forward, too."""
    from crosslayer_transcoder_b200 import fp8

    calls = []
    for name in ("project", "crosslayer_decode", "jump_relu"):
        f = getattr(fp8, name)
        monkeypatch.setattr(fp8, name, lambda *a, f=f, name=name: calls.append(name) or f(*a))
    x = torch.randn(B, L, D)
    for nl, decoder, want in ((ReLU(), Decoder, "project jump_relu project"), (nn.ReLU(), Decoder, "project jump_relu project"),
                              (JumpReLU(0.0, 1.0, L, F), CrosslayerDecoder, "project jump_relu crosslayer_decode"),
                              (PerLayerTopK(k=3), CrosslayerDecoder, "project crosslayer_decode")):
        model = _model(nl, decoder, _Kept)
        model.eight_bit = True
        calls.clear()
        model(x)
        assert calls == want.split()
        if type(nl) is not nn.ReLU:
            nl.register_forward_hook(lambda m, args, out: None)
            calls.clear()
            model(x)
            assert calls == want.split()


@pytest.mark.parametrize("layers, features", [(1, 1), (1, F), (L, 1), (L, F)])
@pytest.mark.parametrize("batch", [1, B])
def test_thresholds_that_broadcast(layers, features, batch):
    """One threshold for all layers or features, as the eager definition takes it: same results, gradients in theta's shape."""
    model = _model(JumpReLU(0.03, 1.0, layers, features))
    x = torch.randn(batch, L, D)
    eager, switched = _both(model, x)
    assert all(torch.equal(a, b) for a, b in zip(eager, switched))
    theta = model.nonlinearity.theta
    if theta.shape[1:] != (L, F):
        seen = []
        theta.register_hook(lambda g: seen.append(g.shape))
        pre = torch.randn(batch, L, F)

        class Keep(torch.autograd.Function):                # thresholds as the operator gets them
            @staticmethod
            def forward(ctx, x, th):
                assert th.shape == (1, L, F)
                return x * (x > th)

            @staticmethod
            def backward(ctx, g):
                return g, torch.ones(1, L, F)

        from crosslayer_transcoder_b200 import fp8

        fp8.jump_relu = lambda x, th, bw: Keep.apply(x, th)  # (put back with the fixture)
        model.nonlinearity(pre, eight_bit=True).sum().backward()
        assert torch.equal(theta.grad, torch.ones(1, L, F).sum_to_size(theta.shape)) and seen == [theta.shape]


def test_thresholds_that_do_not_fit_are_refused():
    with pytest.raises(ValueError):
        JumpReLU(0.03, 1.0, L + 1, F)(torch.randn(B, L, F), eight_bit=True)
