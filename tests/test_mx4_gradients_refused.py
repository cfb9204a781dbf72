"""The MXFP4 calls have no gradient, in either mode: inputs that carry one are refused (on the CPU: the checks alone)."""
import pytest
import torch
from torch.autograd import forward_ad

import llp_hip as K
import llp_mx


@pytest.fixture(autouse=True)
def _checks_alone(monkeypatch):
    monkeypatch.setattr(llp_mx, "_on_gpu", lambda dev: None)
    monkeypatch.setattr(K, "launch", lambda *a: None)


def _w():
    return llp_mx.MX4(torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4, dtype=torch.uint8), 100)


def _calls(x, b):
    return [lambda: llp_mx.quantize(x), lambda: llp_mx.quantize(torch.zeros(2, 100), None, x), lambda: llp_mx.linear(x, _w()),
            lambda: llp_mx.linear(x.view(1, 2, 100), _w()), lambda: llp_mx.linear(torch.zeros(2, 100), _w(), b)]


def test_backward_mode():
    for call in _calls(torch.zeros(2, 100, requires_grad=True), torch.zeros(3, requires_grad=True)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


def test_forward_mode():
    with forward_ad.dual_level():
        for call in _calls(forward_ad.make_dual(torch.zeros(2, 100), torch.ones(2, 100)),
                           forward_ad.make_dual(torch.zeros(3), torch.ones(3))):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with pytest.raises(RuntimeError, match="no gradient"), torch.no_grad():
                call()
        for call in _calls(torch.zeros(2, 100), torch.zeros(3)):
            call()


def test_function_transforms():
    x, w = torch.zeros(2, 100), _w()
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.jvp(lambda y: llp_mx.linear(y, w), (x,), (x,))
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.func.grad(lambda y: llp_mx.linear(y, w).sum())(x)
