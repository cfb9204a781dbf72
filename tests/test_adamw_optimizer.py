"""llp_optim.AdamW's bookkeeping on the CPU: the step's table is a stand-in."""
import pytest
import torch

import llp_hip as K
import llp_optim


class _Table:
    def __init__(self, params, grads):
        self.params, self.grads = params, grads

    def step(self, ctr, **kw):
        self.kw = kw


@pytest.fixture
def tables(monkeypatch):
    """The tables that step() builds, in order; launches are left out but for the step counter's."""
    made = []

    def table(self, params, grads, **more):
        for p in params:
            self.init_state(p)
        made.append(_Table(params, grads))
        return made[-1]
    monkeypatch.setattr(llp_optim.AdamW, "table", table)
    ctrs = {}

    real = torch.zeros

    def zeros(*a, **kw):
        t = real(*a, **kw)
        if kw.get("dtype") == torch.int64:
            ctrs[t.data_ptr()] = t
        return t
    monkeypatch.setattr(llp_optim.torch, "zeros", zeros)
    monkeypatch.setattr(K, "launch", lambda what, dev, at: ctrs[at].add_(1))
    return made


def test_a_gradient_in_another_layout_is_another_table(tables):
    p, g = torch.nn.Parameter(torch.zeros(6, 6)), torch.randn(6, 6)
    opt = llp_optim.AdamW([p])
    p.grad = g
    opt.step(), opt.step()
    assert len(tables) == 1
    p.grad = g.t()                       # the same storage, read in another order
    opt.step()
    assert len(tables) == 2 and not tables[1].grads[0].is_contiguous()      # (the real table refuses it)


@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_state_is_another_table(tables, bits):
    p = torch.nn.Parameter(torch.zeros(6, 6))
    opt = llp_optim.AdamW([p], state_bits=bits)
    p.grad = torch.randn(6, 6)
    opt.step()
    for n, name in enumerate(k for k in list(opt.state[p]) if k != "step"):
        opt.state[p][name] = opt.state[p][name].clone()
        opt.step()
        assert len(tables) == 2 + n, name
        opt.step()
        assert len(tables) == 2 + n, name
    assert float(opt.state_dict()["state"][0]["step"]) == 1 + 2 * (len(opt.state[p]) - 1)
