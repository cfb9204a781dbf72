"""Given negative edges on several ranks: every rank takes its own and counts them all."""
import torch


def test_injected_negatives_count_every_ranks(monkeypatch):
    import llp_engine
    e = llp_engine.EngineBase.__new__(llp_engine.EngineBase)
    e.dev, e.world, e.rank, e.group, e.N = torch.device("cpu"), 2, 0, None, 50
    e._buf = lambda name, shape, dtype: torch.full(shape, -1, dtype=dtype)
    monkeypatch.setattr(llp_engine, "_all_reduce", lambda t, group=None: t.add_(7))      # the other rank's seven
    neg = torch.arange(10).view(2, 5)
    got, n, total, count = e._negatives(8, 16, 0, neg, False)
    assert (n, total, count) == (5, 12, None) and torch.equal(got.long(), neg)
