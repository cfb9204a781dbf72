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


def _mx4(flat, at, rows=10, cols=100, ld_codes=64, ld_scales=4, scales_at=None):
    p = -(-cols // 128) * 128
    scales_at = at + rows * ld_codes if scales_at is None else scales_at
    return llp_mx.MX4(torch.as_strided(flat, (rows, p // 2), (ld_codes, 1), at),
                      torch.as_strided(flat, (rows, p // 32), (ld_scales, 1), scales_at), cols)


def test_mx4_outputs_overlap_no_index():
    flat = torch.zeros(8192, dtype=torch.uint8)
    out, x = _mx4(flat, 0), torch.zeros(20, 100)
    words = flat.view(torch.int32)
    llp_mx._apart("x", out, x, words[170:180].view(1, -1), words[0:0].view(1, -1))
    for idx in (words[0:10], words[155:165], words[165:175]):      # codes, codes and scales, scales
        with pytest.raises(ValueError, match="overlaps"):
            llp_mx._apart("x", out, x, idx.view(1, -1))


def test_quantize_checks_its_indices(monkeypatch):
    """quantize looks at both index tensors (the checks alone: nothing is launched)."""
    monkeypatch.setattr(llp_mx, "_rows2d", lambda x, what: None)
    monkeypatch.setattr(K, "launch", lambda *a: None)
    flat = torch.zeros(8192, dtype=torch.uint8)
    out, x, words = _mx4(flat, 0), torch.zeros(20, 100), flat.view(torch.int32)
    free, bad = words[1000:1010], words[20:30]
    assert llp_mx.quantize(x, free, x, free, out=out) is out
    for i, j in ((bad, free), (free, bad)):
        with pytest.raises(ValueError, match="overlaps"):
            llp_mx.quantize(x, i, x, j, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        llp_mx.quantize(x, bad, out=out)


def test_mx4_codes_and_scales_of_an_output_are_apart():
    flat = torch.zeros(8192, dtype=torch.uint8)
    x = torch.zeros(20, 100)
    llp_mx._apart("x", _mx4(flat, 0, ld_codes=80, ld_scales=80, scales_at=64), x)      # side by side in rows of 80 bytes
    for at in (60, 636):
        with pytest.raises(ValueError, match="codes and scales overlap"):
            llp_mx._apart("x", _mx4(flat, 0, scales_at=at), x)
    row = torch.zeros(1, 100).expand(20, 100)                                          # an input that is one row in memory
    llp_mx._apart("x", _mx4(flat, 0), row)
    llp_mx._apart("x", row, _mx4(flat, 0))                                             # (its own rows: _row_stride)


def test_many_tensors():
    ps = [torch.zeros(2, 4) for _ in range(2000)]
    wide, own = torch.zeros(2, 4 * 100), [torch.zeros(2, 6) for _ in range(1900)]
    copies = [(wide[:, 4 * i:], 4 * 100) for i in range(100)] + [(t, 6) for t in own]
    _apart(ps, copies)
    copies[700] = (own[3].view(-1)[7:], 6)
    with pytest.raises(ValueError, match="overlaps"):
        _apart(ps, copies)
