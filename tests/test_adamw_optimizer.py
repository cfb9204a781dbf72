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
    opt.init_state(p)["note"] = "a user's own entry"
    opt.step()
    del opt.state[p]["note"]
    for n, name in enumerate(k for k in list(opt.state[p]) if k != "step"):
        opt.state[p][name] = opt.state[p][name].clone()
        opt.step()
        assert len(tables) == 2 + n, name
        opt.step()
        assert len(tables) == 2 + n, name
    assert float(opt.state_dict()["state"][0]["step"]) == 1 + 2 * (len(opt.state[p]) - 1)


def _stepped(cls, **kw):
    p = torch.nn.Parameter(torch.randn(4, 3))
    p.grad = torch.randn(4, 3)
    opt = cls([p], **kw)
    opt.step()
    return opt.state_dict()


def test_checkpoints_that_ask_for_more_are_refused():
    p = torch.nn.Parameter(torch.randn(4, 3))
    opt = llp_optim.AdamW([p], lr=0.5)
    for sd, why in ((_stepped(torch.optim.AdamW, amsgrad=True), "amsgrad"), (_stepped(torch.optim.AdamW, maximize=True), "maximize"),
                    (_stepped(torch.optim.Adam, weight_decay=0.1), "decoupled")):
        with pytest.raises(ValueError, match=why):
            opt.load_state_dict(sd)
    eight = llp_optim.AdamW([p], state_bits=8, lr=0.5)
    with pytest.raises(ValueError, match="8 bits"):
        eight.load_state_dict(_stepped(torch.optim.AdamW))
    for o in (opt, eight):               # nothing was taken over
        assert not o.state and o.param_groups[0]["lr"] == 0.5 and "amsgrad" not in o.param_groups[0]
    opt.load_state_dict(_stepped(torch.optim.AdamW, lr=0.25))
    assert opt.param_groups[0]["lr"] == 0.25 and float(opt.state[p]["step"]) == 1
    opt.load_state_dict(_stepped(torch.optim.Adam))      # (no decay: the same update)
    empty = torch.optim.AdamW([p]).state_dict()
    opt.load_state_dict(empty), eight.load_state_dict(empty)


@pytest.mark.parametrize("name", ["amsgrad", "maximize"])
def test_groups_that_ask_for_more_are_refused(name):
    a, b = (torch.nn.Parameter(torch.zeros(3)) for _ in "ab")
    with pytest.raises(ValueError, match=name):
        llp_optim.AdamW([{"params": [a], name: True}])
    opt = llp_optim.AdamW([{"params": [a], name: False}])
    with pytest.raises(ValueError, match=name):
        opt.add_param_group({"params": [b], name: True})
    assert len(opt.param_groups) == 1


def test_a_step_counts_as_a_write_in_place(tables):
    """What a forward saved of a param is out of date after the step: backward raises, as after torch's."""
    w, x = torch.nn.Parameter(torch.randn(3, 3)), torch.randn(3, 3, requires_grad=True)
    loss = (x @ w).sum()
    w.grad = torch.randn(3, 3)
    llp_optim.AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradients_are_not_kept(monkeypatch):
    """zero_grad() lets go of the gradients: the optimizer holds none of them (a captured step's are another matter)."""
    import weakref

    class Grads(list):
        pass
    made = []

    class Table:
        def __init__(self, params, grads, *a, **kw):
            self._grads = Grads(grads)
            made.append(weakref.ref(self._grads))

        def step(self, ctr, **kw):
            pass
    Table.state8 = staticmethod(llp_optim.AdamWTable.state8)
    monkeypatch.setattr(llp_optim, "AdamWTable", Table)
    monkeypatch.setattr(K, "launch", lambda *a: None)
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    opt = llp_optim.AdamW([p])
    opt.step()
    assert len(made) == 1 and made[0]() is None


def test_loaded_second_moments_are_not_0_beside_first_ones():
    p = torch.nn.Parameter(torch.zeros(6))
    opt = llp_optim.AdamW([p], state_bits=8)
    opt.init_state(p)
    sd = opt.state_dict()
    sd["state"][0]["exp_avg"] = torch.tensor([0, 5, 128, 133, 7, 0], dtype=torch.uint8)       # (128: -0)
    sd["state"][0]["exp_avg_sq"] = kept = torch.tensor([0, 0, 0, 0, 9, 4], dtype=torch.uint8)
    opt.load_state_dict(sd)
    assert opt.state[p]["exp_avg_sq"].tolist() == [0, 1, 0, 1, 9, 4] and kept.tolist() == [0, 0, 0, 0, 9, 4]
    assert opt.state[p]["exp_avg"].tolist() == [0, 5, 128, 133, 7, 0]
