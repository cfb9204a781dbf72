"""Refusals and host-side checks of the low-bit operators (llp_mx, llp_optim and their C entries), on the CPU."""
import ctypes as C

import numpy as np
import pytest
import torch

import llp_hip as K
import llp_mx
import llp_optim
from oracle import lowbit_oracle as Q


def _u8(*s):
    return torch.zeros(*s, dtype=torch.uint8)


def test_mx4_object_checks():
    llp_mx.MX4(_u8(3, 64), _u8(3, 4), 100)
    with pytest.raises(TypeError):
        llp_mx.MX4(torch.zeros(3, 64), _u8(3, 4), 100)
    with pytest.raises(ValueError):
        llp_mx.MX4(_u8(3, 64), _u8(3, 4), 129)
    with pytest.raises(ValueError):
        llp_mx.MX4(_u8(3, 64), _u8(2, 4), 100)
    with pytest.raises(ValueError):
        llp_mx.MX4(_u8(64, 3).t(), _u8(3, 4), 100)
    with pytest.raises(ValueError):
        llp_mx.MX4(_u8(3, 0), _u8(3, 0), 0)


def test_mx4_cpu_tensors_and_types_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        llp_mx.quantize(torch.zeros(2, 4))
    with pytest.raises(TypeError):
        llp_mx.quantize(torch.zeros(2, 4, dtype=torch.float64))
    with pytest.raises(ValueError):
        llp_mx.quantize(torch.zeros(4))
    with pytest.raises(ValueError):
        llp_mx.quantize(torch.zeros(4, 2).t())
    w = llp_mx.MX4(_u8(3, 64), _u8(3, 4), 100)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        llp_mx.linear(torch.zeros(2, 100), w)


def _entry(name, *args):
    rc = getattr(K.load(), name)(*args)
    return rc, K.load().llp_last_error().decode()


def test_mx4_c_entries_refuse():
    op = K.Operand(4096, None, None, None, 128, 0, None)
    ok = K.Mx4(4096, 4096, 64, 4)
    for bad, why in ((K.Mx4(4097, 4096, 64, 4), "16-B"), (K.Mx4(4096, 4096, 48, 4), "rows"), (K.Mx4(4096, 4096, 64, 2), "rows"),
                     (K.Mx4(None, 4096, 64, 4), "null"), (K.Mx4(4096, 4098, 64, 4), "4-B"), (K.Mx4(4096, 4096, 72, 4), "16-B")):
        rc, msg = _entry("llp_mx4_quantize", 0, 2, 128, C.byref(op), C.byref(bad), None)
        assert rc == 10001 and why in msg, msg
        rc, msg = _entry("llp_mx4_dequantize", 2, 128, C.byref(bad), 0, 4096, 128, None)
        assert rc == 10001 and why in msg, msg
        rc, msg = _entry("llp_gemm_nt_mx4", 2, 2, 128, 0, None, C.byref(bad), C.byref(ok), 4096, 2, 0, None, None, 0, None)
        assert rc == 10001 and why in msg, msg
    for args, why in (
            ((2, 2, 128, 0, None, None, C.byref(ok), 4096, 2, 0, None, None, 0, None), "one of A"),
            ((2, 2, 128, 0, C.byref(K.Operand(4096, 4096, None, None, 128, 0, None)), C.byref(ok), C.byref(ok), 4096, 2, 0, None,
              None, 0, None), "plain rows"),
            ((2, 2, 128, 0, None, C.byref(ok), C.byref(ok), None, 2, 0, None, None, 0, None), "one of C"),
            ((2, 2, 128, 0, None, C.byref(ok), C.byref(ok), 4096, 2, 0, C.byref(ok), None, 0, None), "one of C"),
            ((2, 2, 128, 0, None, C.byref(ok), C.byref(ok), 4096, 2, 0, None, None, 2, None), "act"),
            ((2, 2, 128, 0, None, C.byref(ok), C.byref(ok), 4096, 1, 0, None, None, 0, None), "overlap"),
            ((2, 2, 128, 2, C.byref(op), None, C.byref(ok), 4096, 2, 0, None, None, 0, None), "f32 or bf16"),
            ((2, 2, 128, 0, None, C.byref(ok), C.byref(ok), 4096, 2, 2, None, None, 0, None), "f32 or bf16"),
            ((2, 2, 0, 0, None, C.byref(ok), C.byref(ok), 4096, 2, 0, None, None, 0, None), "K >= 1"),
            ((-1, 2, 8, 0, None, C.byref(ok), C.byref(ok), 4096, 2, 0, None, None, 0, None), "M, N >= 0")):
        rc, msg = _entry("llp_gemm_nt_mx4", *args)
        assert rc == 10001 and why in msg, (why, msg)
    assert _entry("llp_gemm_nt_mx4", 0, 2, 128, 0, None, C.byref(ok), C.byref(ok), None, 0, 0, None, None, 0, None)[0] == 0
    rows = K.Operand(4096, None, None, None, 128, 0, 4096)
    assert "device row count" in _entry("llp_mx4_quantize", 0, 2, 128, C.byref(rows), C.byref(ok), None)[1]


def test_adamw_c_entries_refuse():
    good = dict(descs=4096, n=1, work=4096, n_work=1, bits=32, pt=0, gt=0, sumsq=None, mn=1.0, lr=0.1, b1=0.9, b2=0.99,
                eps=1e-8, wd=0.0, step=4096, seed=0, stream=None)
    for change, why in (({"bits": 16}, "state_bits"), ({"pt": 2}, "f32 or bf16"), ({"gt": -1}, "f32 or bf16"),
                        ({"lr": -1.0}, "lr"), ({"b1": 1.0}, "betas"), ({"b2": -0.1}, "betas"), ({"wd": -1.0}, "weight_decay"),
                        ({"eps": float("nan")}, "eps"), ({"descs": None}, "null"), ({"work": None}, "null"),
                        ({"step": None}, "null"), ({"n": 70000}, "n_tensors"), ({"n_work": -1}, "n_work")):
        rc, msg = _entry("llp_adamw_step", *{**good, **change}.values())
        assert rc == 10001 and why in msg, (change, msg)
    assert _entry("llp_adamw_step", *{**good, "n_work": 0}.values())[0] == 0
    assert _entry("llp_adamw_values", 4096, 4096, 1, 2, None)[0] == 10001
    assert _entry("llp_adamw_copy_t", None, 4096, 1, 0, None)[0] == 10001
    L = K.load()
    assert [L.llp_adamw_work_items(n) for n in (0, 1, 2048, 2049)] == [0, 1, 1, 2]
    assert L.llp_adamw_copy_t_items(65, 64) == 2


def _lists(n=40):
    f = [torch.zeros(n)]
    return f, [torch.zeros(n)], [torch.zeros(n)], [torch.zeros(n)]


def test_adamw_table_refuses():
    p, g, m, v = _lists()
    T = llp_optim.AdamWTable
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        T(p, g, m, v)
    with pytest.raises(ValueError, match="no params"):
        T([], [], [], [])
    with pytest.raises(ValueError):
        T(p, g + g, m, v)
    with pytest.raises(TypeError):
        T(p, [torch.zeros(40, dtype=torch.float64)], m, v)
    with pytest.raises(TypeError):
        T(p, g, [torch.zeros(40, dtype=torch.bfloat16)], v)
    with pytest.raises(ValueError):
        T(p, [torch.zeros(39)], m, v)
    with pytest.raises(ValueError):
        T([torch.zeros(8, 10)[:, ::2]], g, m, v)
    with pytest.raises(ValueError, match="together"):
        T(p, g, [_u8(40)], [_u8(40)], exp_avg_scale=[_u8(2)])
    with pytest.raises(ValueError, match="exp_avg_scale"):
        T(p, g, [_u8(40)], [_u8(40)], exp_avg_scale=[_u8(1)], exp_avg_sq_scale=[_u8(2)])
    with pytest.raises(ValueError, match="group"):
        T(p, g, m, v, groups=[8])
    with pytest.raises(ValueError, match="out has no"):
        T(p, g, m, v, out={"exp_avg_scale": [_u8(2)]})
    with pytest.raises(ValueError, match="values"):
        T(p, g, m, v, values={"exp_avg": m})


def test_adamw_table_refuses_overlaps():
    flat = torch.zeros(400)
    a, b, c, d = flat[:40], flat[100:140], flat[200:240], flat[300:340]
    apart = llp_optim.AdamWTable._apart
    none = [(None, 0)]

    def ins(p=a, m=c, v=d):
        return {"params": [p], "exp_avg": [m], "exp_avg_sq": [v]}

    apart(ins(), ins(), [b], none, none, None)                                     # in place
    apart(ins(), ins(p=flat[40:80]), [b], none, none, None)                        # beside
    for bad in (ins(p=flat[20:60]), ins(p=b), ins(m=flat[210:250]), ins(v=c)):
        with pytest.raises(ValueError, match="overlaps"):
            apart(ins(), bad, [b], none, none, None)
    with pytest.raises(ValueError, match="overlaps"):                              # the same param twice
        apart({"params": [a, a], "exp_avg": [c, flat[250:290]], "exp_avg_sq": [d, flat[350:390]]},
              {"params": [a, a], "exp_avg": [c, flat[250:290]], "exp_avg_sq": [d, flat[350:390]]}, [b, b], none * 2, none * 2, None)
    with pytest.raises(ValueError, match="overlaps"):                              # a gradient that is the param
        apart(ins(), ins(), [a], none, none, None)
    apart(ins(), ins(), [b], [(flat[140:180], 0)], none, None)
    with pytest.raises(ValueError, match="overlaps"):
        apart(ins(), ins(), [b], [(flat[120:160], 0)], none, None)


def test_adamw_optimizer_refuses():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(lr=-1), dict(betas=(1.0, 0.9)), dict(eps=-1), dict(weight_decay=-1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            llp_optim.AdamW([p], **kw)
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        llp_optim.AdamW([p]).step()


def test_oracle_round_trips():
    """The 64-bit restatement: every code is its own nearest, draws keep the mean, scales hold the block."""
    for signed in (True, False):
        lv = Q.levels8(signed)
        assert (np.diff(lv) > 0).all() and lv[-1] == (448 if signed else 496)
        # over all 65,536 draws the mean is the value, to one draw's share of the codes' distance (1/8)
        for x in np.linspace(1, 1.0625, 9):
            x = np.full(65536, x)
            s = Q.scales8(x, signed)
            c, _ = Q.round8(x if signed else x * x, np.arange(65536), s, signed)
            q = Q.values8(c, s, signed)
            assert abs((q if signed else q * q).mean() - (x[0] if signed else x[0] ** 2)) <= 0.125 / 65536 + 1e-12
    v = np.concatenate([-Q.E2M1[::-1], Q.E2M1])[None, :]
    assert np.array_equal(Q.mx4_round(v), v)
    d = Q.draws16(20, 3, 5, 99)
    from oracle import llp_oracle as O
    assert d[9] == (int(O.philox_u32(99, 65536 * 5 + 3, np.array([4]))[0]) >> 16) & 0xFFFF


def test_adamw_copies_are_bounded():
    """A copy has the param's size, or rows that stay within its storage."""
    fits = llp_optim.AdamWTable._fits
    t = torch.zeros(6, 20)
    fits((None, 0), 3, 4, 0)
    fits((t, 0), 6, 20, 0)
    fits((t, 20), 6, 10, 0)
    fits((t[:, 10:], 20), 6, 10, 0)
    fits((t[5:], 20), 1, 20, 0)
    for copy, r, c in (((t, 0), 6, 19), ((t, 20), 7, 20), ((t[:, 11:], 20), 6, 10), ((t, 8), 6, 10), ((t[1:], 20), 6, 20)):
        with pytest.raises(ValueError):
            fits(copy, r, c, 0)
    p, g, m, v = [[torch.zeros(6, 20)] for _ in range(4)]
    with pytest.raises(ValueError, match="copy"):
        llp_optim.AdamWTable(p, g, m, v, copies=[torch.zeros(6, 19)])
    with pytest.raises(ValueError, match="copy"):
        llp_optim.AdamWTable(p, g, m, v, copies_t=[(torch.zeros(20, 5), 6)])


def test_mx4_on_the_cpu_is_refused():
    q = llp_mx.MX4(_u8(3, 64), _u8(3, 4), 100)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        llp_mx.dequantize(q)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        llp_mx.linear(q, q)


def test_commands_optimizer_flags():
    import main
    import train_teacher_gnn
    for mod in (main, train_teacher_gnn):
        a = mod.build_parser().parse_args([])
        assert (a.optimizer, a.weight_decay, a.optim_bits) == ("adam", 0.01, 32)
        p = [torch.nn.Parameter(torch.zeros(3))]
        assert type(llp_optim.from_args(a, p)) is torch.optim.Adam
        a = mod.build_parser().parse_args(["--optimizer=adamw", "--optim_bits=8", "--weight_decay=0.5", "--lr=0.25"])
        opt = llp_optim.from_args(a, p)
        assert isinstance(opt, llp_optim.AdamW) and opt.state_bits == 8
        assert (opt.param_groups[0]["lr"], opt.param_groups[0]["weight_decay"]) == (0.25, 0.5)
        with pytest.raises(ValueError, match="adamw"):
            llp_optim.from_args(mod.build_parser().parse_args(["--optim_bits=8"]), p)
    assert main.build_parser().parse_args([]).eval_dtype == "fp32"


def test_adamw_optimizer_copies():
    """copy.deepcopy (as pickling) keeps the settings and starts with no device tables."""
    import copy
    opt = llp_optim.AdamW([torch.nn.Parameter(torch.zeros(4))], lr=0.5, state_bits=8, seed=9)
    got = copy.deepcopy(opt)
    assert (got.state_bits, got.seed, got.param_groups[0]["lr"], got._tables) == (8, 9, 0.5, {})


def test_mx4_overlaps_are_found():
    flat = torch.zeros(4096, dtype=torch.uint8)
    a = llp_mx.MX4(flat[:640].view(10, 64), flat[640:680].view(10, 4), 100)
    b = llp_mx.MX4(flat[1024:1664].view(10, 64), flat[1664:1704].view(10, 4), 100)
    llp_mx._apart("x", a, b)
    x = flat[2048:].view(torch.float32).view(4, 128)
    llp_mx._apart("x", a, x, b)
    llp_mx._apart("x", a, llp_mx.MX4(_u8(0, 64), _u8(0, 4), 100))
    for bad in (a, llp_mx.MX4(flat[576:1216].view(10, 64), flat[1664:1704].view(10, 4), 100),
                llp_mx.MX4(flat[1024:1664].view(10, 64), flat[676:716].view(10, 4), 100),
                flat[:1024].view(torch.float32).view(2, 128), flat[:640].view(torch.bfloat16).view(10, 32)[:, 8:]):
        with pytest.raises(ValueError, match="overlaps"):
            llp_mx._apart("x", a, bad)


def test_mx4_of_one_row_has_no_stride():
    q = llp_mx.MX4(_u8(5, 64)[2:3], _u8(5, 4).expand(5, 4)[2:3].as_strided((1, 4), (999, 1)), 100)
    assert (q.c.ld_codes, q.c.ld_scales) == (64, 4)


def test_rows_of_a_given_output_do_not_overlap():
    assert llp_mx._row_stride(torch.zeros(4, 12)[:, :10], "x") == 12
    assert llp_mx._row_stride(torch.zeros(1, 10).as_strided((1, 10), (3, 1)), "x") == 10
    for bad in (torch.zeros(1, 10).expand(4, 10), torch.zeros(100).as_strided((4, 10), (9, 1))):
        with pytest.raises(ValueError, match="overlap"):
            llp_mx._row_stride(bad, "x")


def test_adamw_work_pairs():
    assert llp_optim._pairs([2, 0, 3, 0, 1, 2]).tolist() == [[0, 0], [0, 1], [2, 0], [2, 1], [2, 2], [1, 0], [2, 0], [2, 1]]
    assert llp_optim._pairs([0, 0]).shape == (0, 2)
