"""Which buffers of a low-bit call may share memory (host-side checks of llp_optim and llp_mx, on the CPU)."""
import itertools
import random

import pytest
import torch

import llp_hip as K
import llp_mx
import llp_optim


def test_rows_meet_as_sets_of_bytes():
    rng = random.Random(1)

    def rows():
        w = rng.randint(0, 6)
        return rng.randint(0, 60), rng.randint(0, 5), max(w + rng.choice([0, 0, 1, 2, 3, 6]), 1), w

    def bytes_of(r):
        return {r[0] + i * r[2] + j for i in range(r[1]) for j in range(r[3])}

    met = 0
    for _ in range(20000):
        a, b = rows(), rows()
        if rng.random() < 0.4:
            b = (b[0], b[1], max(a[2], b[3], 1), b[3])      # often the same stride
        want = bool(bytes_of(a) & bytes_of(b))
        assert K.rows_meet(a, b) == K.rows_meet(b, a) == want, (a, b)
        met += want
    assert 2000 < met < 18000


def _apart(p, copies, copies_t=None, **more):
    flat = torch.zeros(4 * sum(t.numel() for t in p) + 64)
    at = itertools.accumulate([0] + [t.numel() for t in p * 3])
    rest = [flat[o:o + t.numel()] for o, t in zip(at, p * 3)]
    n = len(p)
    ins = {"params": p, "exp_avg": more.get("m", rest[:n]), "exp_avg_sq": rest[n:2 * n]}
    llp_optim.AdamWTable._apart(ins, ins, more.get("g", rest[2 * n:]), copies, copies_t or [(None, 0)] * n, None)


def test_strided_copies_that_overlap_are_refused():
    w = torch.zeros(6, 20)
    p = torch.zeros(6, 8)
    none = (None, 0)
    _apart([p], [(w, 20)])
    for bad in ((p, 8), (p.view(-1)[4:], 8), (p, 10)):                       # the param itself
        with pytest.raises(ValueError, match="overlaps"):
            _apart([p], [bad])
    with pytest.raises(ValueError, match="overlaps"):                        # a gradient in the copy's rows
        _apart([p], [(w, 20)], g=[w.view(-1)[60:108]])
    with pytest.raises(ValueError, match="overlaps"):                        # a moment
        _apart([p], [(w, 20)], m=[w.view(-1)[:48]])
    # side by side in one operand, as [Wl | Wr], and its transpose
    q, wt = torch.zeros(6, 12), torch.zeros(20, 6)
    _apart([p, q], [(w, 20), (w[:, 8:], 20)], [(wt, 6), (wt[8:], 6)])
    with pytest.raises(ValueError, match="overlaps"):
        _apart([p, q], [(w, 20), (w[:, 7:], 20)])
    with pytest.raises(ValueError, match="overlaps"):
        _apart([p, q], [(w, 20), none], [none, (w.view(-1), 20)])
    with pytest.raises(ValueError, match="overlaps"):                        # other strides
        _apart([p, q], [(w, 20), (torch.as_strided(w, (6, 12), (13, 1), 19), 13)])
    # a bias in the columns that no copy takes: beside them
    wide = torch.zeros(2, 20)
    _apart([torch.zeros(2, 8), wide[0, 8:20]], [(wide, 20), none])
    with pytest.raises(ValueError, match="overlaps"):
        _apart([torch.zeros(2, 8), wide[0, 7:19]], [(wide, 20), none])


def test_many_tensors():
    ps = [torch.zeros(2, 4) for _ in range(2000)]
    wide, own = torch.zeros(2, 4 * 100), [torch.zeros(2, 6) for _ in range(1900)]
    copies = [(wide[:, 4 * i:], 4 * 100) for i in range(100)] + [(t, 6) for t in own]
    _apart(ps, copies)
    copies[700] = (own[3].view(-1)[7:], 6)
    with pytest.raises(ValueError, match="overlaps"):
        _apart(ps, copies)
