"""What autograd may do with results of the 8-bit passes, on the CPU: a library that launches nothing in place of the kernels."""
import pytest
import torch

from crosslayer_transcoder_b200 import fp8


class _Nothing:
    def call(self, name, *args):
        pass

    def query(self, name, *args):
        return 1


@pytest.fixture(autouse=True)
def _no_library(monkeypatch):
    monkeypatch.setattr(fp8, "lib", _Nothing)
    monkeypatch.setattr(fp8, "_on", lambda device, fn, *args: fn(*args))
    monkeypatch.setattr(fp8, "_status_word", lambda: None)
    monkeypatch.setattr(fp8, "stream_ptr", lambda: 0)


@pytest.mark.parametrize("call", [
    lambda x: fp8.project(x(4, 5, 6), x(6, 7)),
    lambda x: fp8.project(x(4, 6), x(6, 7)),
    lambda x: fp8.project(x(6), x(6, 7), x(7)),
    lambda x: fp8.project(x(4, 3, 6), x(3, 6, 7), x(3, 7)),
    lambda x: fp8.project(x(2, 4, 3, 6), x(3, 6, 7)),
    lambda x: fp8.project(x(3, 6), x(3, 6, 7)),
    lambda x: fp8.project(x(0, 3, 6), x(3, 6, 7)),
    lambda x: fp8.crosslayer_decode(x(4, 2, 6), [x(1, 6, 7), x(2, 6, 7)]),
    lambda x: fp8.crosslayer_decode(x(5, 4, 2, 6), [x(1, 6, 7), x(2, 6, 7)], x(2, 7)),
    lambda x: fp8.crosslayer_decode(x(2, 6), [x(1, 6, 7), x(2, 6, 7)]),
    lambda x: fp8.jump_relu(x(4, 5, 6), x(5, 6)),
])
def test_results_may_be_changed_in_place(call):
    """A bias that is added in place, an in-place nonlinearity."""
    leaves = []

    def leaf(*shape):
        leaves.append(torch.zeros(shape, requires_grad=True))
        return leaves[-1]

    y = call(leaf)
    shape = y.shape
    y.mul_(2.0)
    assert y.shape == shape and y.shape[:-1] == leaves[0].shape[:-1] and y.is_contiguous()
    y.sum().backward()
    assert all(t.grad.shape == t.shape for t in leaves)


def test_thresholds_without_a_gradient_are_not_kept():
    """x's gradient takes the two bits alone: such thresholds and the bandwidth may change, or be inference tensors."""
    with torch.inference_mode():
        frozen = torch.zeros(7)
    for theta in (torch.zeros(7), frozen):
        x, bandwidth = torch.zeros(4, 7, requires_grad=True), torch.ones(())
        y = fp8.jump_relu(x, theta, bandwidth)
        if theta is not frozen:
            theta.add_(1.0)
        bandwidth.mul_(0.5)
        y.sum().backward()
        assert x.grad.shape == x.shape
    x, theta = torch.zeros(4, 7, requires_grad=True), torch.zeros(7, requires_grad=True)
    y = fp8.jump_relu(x, theta, bandwidth)
    bandwidth.mul_(0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):     # the thresholds' gradient does take it
        y.sum().backward()
