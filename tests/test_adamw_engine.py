"""What the training engines take from llp_optim.AdamW, on the CPU: the step and the norm are stand-ins."""
import types

import pytest
import torch

import llp_engine
import llp_hip as K
import llp_optim


def _engine(opt, params, seed=5):
    e = llp_engine.EngineBase.__new__(llp_engine.EngineBase)
    e.dev, e.world, e.seed, e.optimizer, e.all_params = torch.device("cpu"), 1, seed, opt, params
    return e


def test_the_optimizers_seed_counts(monkeypatch):
    monkeypatch.setattr(K, "grad_sumsq", lambda *a, **kw: None)
    ps = [torch.nn.Parameter(torch.zeros(4))]
    seeds = []
    for engine, opt in ((5, 0), (5, 1), (6, 0), (5, 7919)):
        e = _engine(llp_optim.AdamW(ps, state_bits=8, seed=opt), ps, engine)
        e.descs_dev = e.n_desc = e.max_numel = e.n_groups = e.sumsq = e.ws_sumsq = e.sumsq_ticket = e.n_work_sumsq = e.adam_step = None
        e.adamw = types.SimpleNamespace(step=lambda ctr, seed, **kw: seeds.append(seed))
        e._allreduce_and_update()
    assert len(set(seeds)) == 4 and seeds[0] == 5 ^ llp_engine._ADAMW_KEY


def test_params_of_different_age_are_refused():
    ps = [torch.nn.Parameter(torch.zeros(4)) for _ in range(3)]
    opt = llp_optim.AdamW(ps)
    for p in ps:
        opt.init_state(p)["step"] = torch.tensor(4.0)
    e = _engine(opt, ps)
    e._init_optimizer_state()
    assert int(e.adam_step) == 4
    opt.state[ps[0]]["step"] = torch.tensor(3.0)
    with pytest.raises(ValueError, match="same number of steps"):
        e._init_optimizer_state()
