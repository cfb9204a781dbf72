"""AdamW over many tensors (csrc/adamw.hip, llp_optim) against the formulas in 64 bits.

Tolerances: u = 2^-24 is the largest relative error of one f32 rounding (bf16: 2^-8).
  coefficient c of a clipped gradient: a root, a sum, a division: 3 u.
  m' = b1 m + c1 (c g): the constants, both products, c, the sum: at most 8 u (|b1 m| + |c1 c g|).
  v' likewise: c twice, both products with it, the constants, the sum: at most 13 u v'.
  p': keep p: 2 u |p|; the update: m' (8 u of its terms), the root of v' (7.5 u), 1 / sqrt(1 - b2^t), its
  product, eps and the sum (4 u), the division, size and its product (3 u): at most 24 u of
  size (|b1 m| + |c1 c g|) / denominator; the difference: 1 u.
"""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as Q

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
HYPER = dict(lr=0.01, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def _opt():
    import llp_optim
    return llp_optim


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _problem(sizes, seed, bits=32, ptype=torch.float32, gtype=torch.float32, offset=0):
    """Lists p, g, m, v (values for 32 bits; codes and scales for 8) in flat buffers that begin `offset`
    elements late, so that tensors sit at odd addresses."""
    gen = torch.Generator().manual_seed(seed)
    P, G, M, V, MS, VS = [], [], [], [], [], []

    def at(t, dtype):
        flat = torch.zeros(t.numel() + offset, dtype=dtype, device=DEV)
        flat[offset:] = t.reshape(-1).to(dtype)
        return flat[offset:].view(t.shape)

    for i, s in enumerate(sizes):
        size = 1e-3 * torch.exp(torch.randn(s, generator=gen))
        P.append(at(0.1 * torch.randn(s, generator=gen), ptype))
        G.append(at(torch.randn(s, generator=gen) * size, gtype))
        m, r = 0.3 * torch.randn(s, generator=gen) * size, size
        if bits == 32:
            M.append(at(m, torch.float32))
            V.append(at(r * r, torch.float32))
        else:
            for x, signed, codes, scales in ((m, True, M, MS), (r, False, V, VS)):
                x = x.reshape(-1).double().numpy()
                b = Q.scales8(np.abs(x), signed)
                # nearest below: the middle draw of the lower code
                c, _ = Q.round8(x if signed else x * x, np.full(x.size, 0xFFFF), b, signed)
                codes.append(at(torch.from_numpy(c), torch.uint8))
                scales.append(at(torch.from_numpy(b), torch.uint8))
    return P, G, M, V, MS, VS


SIZES = [
    [(1,)],
    [(31,), (32,), (33,), (0,), (7,), (8,), (9,)],
    [(2047,), (2048,), (2049,), (64, 65), (3, 5, 7)],
    [(301, 517), (517,), (1, 517), (1,)],
    [(1 << 20) + 13],
]


def _shapes(sizes):
    return [s if isinstance(s, tuple) else (s,) for s in sizes]


@pytest.mark.parametrize("sizes", range(len(SIZES)))
@pytest.mark.parametrize("ptype,gtype", [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "float32"),
                                         ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("step,clip,offset", [(0, False, 0), (1234, True, 3)])
def test_adamw_f32_moments(sizes, ptype, gtype, step, clip, offset):
    o = _opt()
    pt, gt = getattr(torch, ptype), getattr(torch, gtype)
    P, G, M, V, _, _ = _problem(_shapes(SIZES[sizes]), 10 * sizes + step, ptype=pt, gtype=gt, offset=offset)
    if step == 0:
        for t in M + V:
            t.zero_()
    before = [[_f64(t) for t in ts] for ts in (P, G, M, V)]
    groups = [i % 2 for i in range(len(P))]
    sumsq = torch.tensor([2.5, 0.25], device=DEV) if clip else None
    ctr = torch.full((1,), step, dtype=torch.int64, device=DEV)
    o.AdamWTable(P, G, M, V, groups=groups).step(ctr, sumsq=sumsq, **HYPER)
    assert int(ctr) == step
    for i in range(len(P)):
        p, g, m, v = (b[i] for b in before)
        ss = None if sumsq is None else float(sumsq[groups[i]])
        rp, rm, rv = Q.adamw(p, g, m, v, step + 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], ss)
        c = 1.0 if ss is None else min(1.0, 1.0 / (np.sqrt(ss) + 1e-6))
        terms = 0.9 * np.abs(m) + 0.1 * c * np.abs(g)
        upd = HYPER["lr"] / (1 - 0.9 ** (step + 1)) * terms / (np.sqrt(rv) / np.sqrt(1 - 0.999 ** (step + 1)) + 1e-8)
        assert (np.abs(_f64(M[i]) - rm) <= 8 * U * terms).all()
        assert (np.abs(_f64(V[i]) - rv) <= 13 * U * rv).all()
        tol = 3 * U * np.abs(p) + 24 * U * upd
        if pt == torch.bfloat16:
            tol = tol + 2.0 ** -8 * np.abs(rp)
        assert (np.abs(_f64(P[i]) - rp) <= tol).all()
        assert np.array_equal(_f64(G[i]), g)        # the gradient is not rewritten


@pytest.mark.parametrize("sizes", range(len(SIZES)))
@pytest.mark.parametrize("gtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("step,offset", [(0, 0), (977, 1)])
def test_adamw_8bit_moments(sizes, gtype, step, offset):
    """Every code is the one the draw picks between the codes around the exact value, except where the
    draw lies within the f32 error of the border."""
    o = _opt()
    P, G, M, V, MS, VS = _problem(_shapes(SIZES[sizes]), 7 * sizes + step, bits=8, gtype=getattr(torch, gtype), offset=offset)
    if step == 0:
        for t in M + V + MS + VS:
            t.zero_()
    before = [[t.cpu().numpy().reshape(-1) for t in ts] for ts in (M, MS, V, VS)]
    p0, g0 = [_f64(t).reshape(-1) for t in P], [_f64(t).reshape(-1) for t in G]
    vals = {k: [torch.empty(t.numel(), device=DEV) for t in P] for k in ("exp_avg", "exp_avg_sq")}
    seed = 0x1234567_89ABCDEF
    sumsq = torch.tensor([4.0], device=DEV)
    tab = o.AdamWTable(P, G, M, V, exp_avg_scale=MS, exp_avg_sq_scale=VS, values=vals)
    tab.step(torch.full((1,), step, dtype=torch.int64, device=DEV), sumsq=sumsq, seed=seed, **HYPER)
    tab.values()
    for i in range(len(P)):
        n = p0[i].size
        if n == 0:
            continue
        m0, r0 = Q.values8(before[0][i], before[1][i], True), Q.values8(before[2][i], before[3][i], False)
        rp, rm, rv = Q.adamw(p0[i], g0[i], m0, r0 * r0, step + 1, HYPER["lr"], HYPER["betas"], HYPER["eps"],
                             HYPER["weight_decay"], 4.0)
        c = 1.0 / (2.0 + 1e-6)
        terms = 0.9 * np.abs(m0) + 0.1 * c * np.abs(g0[i])
        upd = HYPER["lr"] / (1 - 0.9 ** (step + 1)) * terms / (np.sqrt(rv) / np.sqrt(1 - 0.999 ** (step + 1)) + 1e-8)
        assert (np.abs(_f64(P[i]).reshape(-1) - rp) <= 3 * U * np.abs(p0[i]) + 24 * U * upd).all()
        w = Q.draws16(n, i, step + 1, seed)
        for x, err, signed, codes, scales, val in (
                (rm, 8 * U * terms, True, M[i], MS[i], vals["exp_avg"][i]),
                (rv, 13 * U * rv, False, V[i], VS[i], vals["exp_avg_sq"][i])):
            got, s = codes.cpu().numpy().reshape(-1), scales.cpu().numpy().reshape(-1)
            size = np.abs(x) if signed else np.sqrt(x)
            lo, hi = Q.scales8(size * (1 - 16 * U), signed), Q.scales8(size * (1 + 16 * U), signed)
            assert ((s == lo) | (s == hi)).all()
            want, room = Q.round8(x, w, s, signed)
            lv = Q.levels8(signed) if signed else Q.levels8(False) ** 2
            f = np.repeat(np.exp2(s.astype(np.float64) - 127), 32)[:n]
            y = np.abs(x) / (f if signed else f * f)
            j = np.clip(np.searchsorted(lv, y, side="right") - 1, 0, lv.size - 2)
            gap = lv[j + 1] - lv[j]
            # below 2^-6 the kernel adds 2^-6 first: another u 2^-6 there; the product u den: 2 u of den
            off = err / (f if signed else f * f) / gap + (U * 2.0 ** -5 / gap if signed else 0) + 4 * U
            near = (room <= off) | (np.minimum(y - lv[j], lv[j + 1] - y) <= off * gap)
            assert ((got & 127 if signed else got)[~near] == (want & 127 if signed else want)[~near]).all()
            # few are near, for gradients of 24 bits: a draw or a value falls within `off` of a border for a share
            # of about 4 off, and off is under 2^-10 but for the smallest codes.  A bf16 gradient times c = 0.5 (1 -
            # 5e-7) and the old code times 0.9 have so few bits that their sum often lies 5e-7 beside a code.
            assert gtype == "bfloat16" or near.mean() < 0.01 or n < 1000
            v = Q.values8(got, s, signed)
            assert np.array_equal(_f64(val), (v if signed else v * v).astype(np.float32).astype(np.float64))


def test_adamw_out_of_place_keeps_the_inputs():
    o = _opt()
    sizes = [(100, 33), (33,), (5000,)]
    P, G, M, V, MS, VS = _problem(sizes, 3, bits=8)
    kept = [[t.clone() for t in ts] for ts in (P, G, M, V, MS, VS)]
    out = {k: [torch.full_like(t, 99) for t in ts] for k, ts in
           (("params", P), ("exp_avg", M), ("exp_avg_sq", V), ("exp_avg_scale", MS), ("exp_avg_sq_scale", VS))}
    ctr = torch.full((1,), 5, dtype=torch.int64, device=DEV)
    o.AdamWTable(P, G, M, V, MS, VS, out=out).step(ctr, seed=4, **HYPER)
    for ts, ks in zip((P, G, M, V, MS, VS), kept):
        assert all(torch.equal(a, b) for a, b in zip(ts, ks))
    o.AdamWTable(P, G, M, V, MS, VS).step(ctr, seed=4, **HYPER)       # in place: the same bits
    for k, ts in (("params", P), ("exp_avg", M), ("exp_avg_sq", V), ("exp_avg_scale", MS), ("exp_avg_sq_scale", VS)):
        assert all(torch.equal(a, b) for a, b in zip(out[k], ts)), k


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_copies(bits):
    """Working copies: the param's shape, rows inside a wider operand, transposed; what lies beside them stays."""
    o = _opt()
    sizes = [(70, 130), (65, 64), (64,), (33, 7)]
    P, G, M, V, MS, VS = _problem(sizes, 8, bits=bits)
    wide = torch.full((70, 200), 7.0, dtype=torch.bfloat16, device=DEV)
    tall = torch.full((130, 80), 7.0, dtype=torch.bfloat16, device=DEV)
    c1, t1 = torch.empty(65, 64, device=DEV), torch.empty(64, 65, device=DEV)
    kw = dict(exp_avg_scale=MS, exp_avg_sq_scale=VS) if bits == 8 else {}
    c2 = torch.empty(64, dtype=torch.bfloat16, device=DEV)
    tab = o.AdamWTable(P, G, M, V, copies=[(wide[:, 10:140], 200), c1, c2, None],
                       copies_t=[(tall[:, 5:75], 80), t1, None, None], **kw)
    tab.step(torch.zeros(1, dtype=torch.int64, device=DEV), **HYPER)
    assert torch.equal(wide[:, 10:140], P[0].bfloat16()) and torch.equal(tall[:, 5:75], P[0].t().bfloat16())
    assert (wide[:, :10] == 7).all() and (wide[:, 140:] == 7).all() and (tall[:, :5] == 7).all() and (tall[:, 75:] == 7).all()
    assert torch.equal(c1, P[1]) and torch.equal(t1, P[1].t()) and torch.equal(c2, P[2].bfloat16())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_nan_and_inf(bits):
    """A NaN gradient makes its element NaN (its block's moments, in 8 bits) and no other; a NaN norm all."""
    o = _opt()
    P, G, M, V, MS, VS = _problem([(200,)], 5, bits=bits)
    kw = dict(exp_avg_scale=MS, exp_avg_sq_scale=VS) if bits == 8 else {}
    G[0][70] = float("nan")
    G[0][150] = float("inf")
    vals = {k: [torch.empty(200, device=DEV)] for k in ("exp_avg", "exp_avg_sq")} if bits == 8 else None
    tab = o.AdamWTable(P, G, M, V, values=vals, **kw)
    ctr = torch.full((1,), 9, dtype=torch.int64, device=DEV)
    tab.step(ctr, **HYPER)
    bad = ~torch.isfinite(P[0])
    assert bad.nonzero().flatten().tolist() == [70, 150]
    if bits == 8:
        tab.values()
        want = torch.zeros(200, dtype=torch.bool, device=DEV)
        want[64:96] = want[128:160] = True
        assert torch.equal(torch.isnan(vals["exp_avg"][0]), want) and torch.equal(torch.isnan(vals["exp_avg_sq"][0]), want)
    else:
        assert torch.equal(~torch.isfinite(M[0]), bad) and torch.equal(~torch.isfinite(V[0]), bad)
    tab.step(ctr, sumsq=torch.full((1,), float("nan"), device=DEV), **HYPER)
    assert torch.isnan(P[0]).all()


def test_adamw_extreme_magnitudes():
    """Moments from the smallest to the largest f32 roots, zero blocks, and blocks of one large value."""
    o = _opt()
    n = 32 * 9
    g = torch.zeros(n)
    for b, e in enumerate([-60, -40, -19, -6, 0, 6, 18]):
        g[32 * b:32 * b + 32] = torch.randn(32, generator=torch.Generator().manual_seed(b)) * 10.0 ** e if e > -38 else 0
    g[32 * 7] = 1e10
    P, G = [torch.zeros(n, device=DEV)], [g.to(DEV)]
    (m, ms), (v, vs) = o.AdamWTable.state8(n, DEV), o.AdamWTable.state8(n, DEV)
    vals = {k: [torch.empty(n, device=DEV)] for k in ("exp_avg", "exp_avg_sq")}
    tab = o.AdamWTable(P, G, [m], [v], [ms], [vs], values=vals)
    tab.step(torch.zeros(1, dtype=torch.int64, device=DEV), lr=0.01, weight_decay=0.0)
    tab.values()
    gm, gv = _f64(vals["exp_avg"][0]), _f64(vals["exp_avg_sq"][0])
    gd = g.double().numpy()
    # between neighbouring codes: E4M3 within 2^-3 of the value, or the block's 2^-9 unit; v within (1 + 2^-4)^2 - 1
    unit = np.repeat(np.exp2(ms.cpu().numpy().astype(np.float64) - 127), 32)
    assert (np.abs(gm - 0.1 * gd) <= np.maximum(2.0 ** -3 * np.abs(0.1 * gd), 2.0 ** -9 * unit) * 1.0001).all()
    rv = 0.001 * gd * gd
    f32 = rv > 2.0 ** -100      # below, v itself leaves f32's normal range
    unit = np.repeat(np.exp2(vs.cpu().numpy().astype(np.float64) - 127), 32)
    q = 2.0 ** -10 * unit       # a code's distance at the bottom: (r + q)^2 - r^2 there
    assert (np.abs(gv - rv) <= 0.13 * rv + 2 * np.sqrt(rv) * q + q * q)[f32].all()
    assert torch.isfinite(P[0]).all()
    assert (gm[gd == 0] == 0).all() and (gv[gd == 0] == 0).all()


def test_adamw_8bit_rounding_keeps_the_mean():
    """Steps with a zero gradient: the moments decay by b1 and b2 in the mean.  Per element the mean of
    m_T over n elements is within 6 standard errors, the variance of one rounding being at most
    (gap / 2)^2 and a later step only shrinking it."""
    o = _opt()
    n, T = 1 << 18, 12
    b1, b2 = 0.9, 0.999
    gen = torch.Generator().manual_seed(0)
    x = 1 + torch.rand(n, generator=gen).double().numpy()
    (m, ms), (v, vs) = o.AdamWTable.state8(n, DEV), o.AdamWTable.state8(n, DEV)
    s = Q.scales8(x, True)
    mc, _ = Q.round8(x, np.full(n, 0xFFFF), s, True)
    sv = Q.scales8(x, False)
    vc, _ = Q.round8(x * x, np.full(n, 0xFFFF), sv, False)
    for t, a in ((m, mc), (ms, s), (v, vc), (vs, sv)):
        t.copy_(torch.from_numpy(a))
    m0, v0 = Q.values8(mc, s, True), Q.values8(vc, sv, False) ** 2
    vals = {k: [torch.empty(n, device=DEV)] for k in ("exp_avg", "exp_avg_sq")}
    tab = o.AdamWTable([torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)], [m], [v], [ms], [vs], values=vals)
    for t in range(T):
        tab.step(torch.full((1,), t, dtype=torch.int64, device=DEV), betas=(b1, b2), seed=77)
    tab.values()
    gm, gv = _f64(vals["exp_avg"][0]), _f64(vals["exp_avg_sq"][0])
    # m <= 2: gaps <= 1/8, T roundings: variance <= T / 256; v <= 4: gaps <= 1/4: variance <= T / 64
    assert abs(gm.mean() - m0.mean() * b1 ** T) <= 6 * np.sqrt(T / 256 / n) + 1e-5
    assert abs(gv.mean() - v0.mean() * b2 ** T) <= 6 * np.sqrt(T / 64 / n) + 1e-5


def test_adamw_replays_in_a_graph():
    """Captured once, replayed with other work between: each replay as the eager step."""
    import llp_hip as K
    o = _opt()
    sizes = [(300, 70), (300,)]
    A, B = _problem(sizes, 2, bits=8), _problem(sizes, 2, bits=8)
    ctrs = [torch.zeros(1, dtype=torch.int64, device=DEV) for _ in "ab"]
    tabs = [o.AdamWTable(*X) for X in (A, B)]

    def one(tab, ctr):
        tab.step(ctr, seed=5, **HYPER)
        K.increment(ctr)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            one(tabs[0], ctrs[0])
    torch.cuda.synchronize()
    for k in range(4):
        graph.replay()
        one(tabs[1], ctrs[1])
        torch.cuda.synchronize()
        for x, y in zip(A, B):
            assert all(torch.equal(a, b) for a, b in zip(x, y)), k
        for X in (A, B):
            for g in X[1]:
                g.mul_(-0.7)


def test_optimizer_matches_torch_adamw():
    """llp_optim.AdamW (32 bits) against torch.optim.AdamW in 64 bits over steps: a step's update is off by
    24 u of its terms plus what m carries over (8 u a step, decaying by 0.9: 80 u), under 200 u; errors add up."""
    o = _opt()
    gen = torch.Generator().manual_seed(4)
    shapes = [(40, 33), (33,), (1,)]
    init = [torch.randn(s, generator=gen) for s in shapes]
    mine = [torch.nn.Parameter(t.to(DEV)) for t in init]
    ref = [torch.nn.Parameter(t.double()) for t in init]
    a = o.AdamW([{"params": mine[:1]}, {"params": mine[1:], "weight_decay": 0.0}], lr=0.02, weight_decay=0.1)
    b = torch.optim.AdamW([{"params": ref[:1]}, {"params": ref[1:], "weight_decay": 0.0}], lr=0.02, weight_decay=0.1)
    T = 10
    for t in range(T):
        for x, y in zip(mine, ref):
            g = torch.randn(x.shape, generator=gen)
            x.grad, y.grad = g.to(DEV), g.double()
        if t == 5:      # saved and loaded half way
            sd = a.state_dict()
            a = o.AdamW([{"params": mine[:1]}, {"params": mine[1:], "weight_decay": 0.0}], lr=0.02, weight_decay=0.1)
            a.load_state_dict(sd)
        a.step()
        b.step()
    # |m'| / sqrt(v') corrected is at most 3.2 and its terms sum to at most 7 of it; T steps
    for x, y in zip(mine, ref):
        tol = T * (4 * U * (y.detach().abs() + 0.02 * T * 4) + 200 * U * 0.02 * 7)
        assert ((x.detach().cpu().double() - y.detach()).abs() <= tol).all()
    assert float(a.state_dict()["state"][0]["step"]) == T


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_dict_round_trip(bits):
    o = _opt()
    gen = torch.Generator().manual_seed(6)
    w0 = torch.randn(50, 41, generator=gen)
    gs = [torch.randn(50, 41, generator=gen).to(DEV) for _ in range(6)]

    def run(reload_at):
        p = torch.nn.Parameter(w0.to(DEV))
        opt = o.AdamW([p], lr=0.01, state_bits=bits, seed=3)
        for t, g in enumerate(gs):
            if t == reload_at:
                sd = opt.state_dict()
                opt = o.AdamW([p], lr=0.01, state_bits=bits, seed=3)
                opt.load_state_dict(sd)
            p.grad = g.clone()
            opt.step()
        return p.detach().clone(), opt.state_dict()["state"][0]

    (p1, s1), (p2, s2) = run(None), run(3)
    assert torch.equal(p1, p2)
    for k in s1:
        assert torch.equal(s1[k], s2[k]), k


def test_optimizer_uses_the_current_stream():
    o = _opt()
    p = torch.nn.Parameter(torch.ones(1 << 22, device=DEV))
    opt = o.AdamW([p], lr=0.5, weight_decay=0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.zeros_like(p)
        for _ in range(20):
            g += 1.0
        p.grad = g
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.allclose(p, torch.full_like(p, 0.5), atol=1e-5)


def test_adamw_8bit_large_tensor():
    """Past 32 M elements the step streams; p, the codes and what lies around a slice of the tensor."""
    o = _opt()
    n = (1 << 25) + 45
    gen = torch.Generator(device=DEV).manual_seed(12)
    p = torch.randn(n, device=DEV, generator=gen)
    g = 1e-3 * torch.randn(n, device=DEV, generator=gen)
    (m, ms), (v, vs) = o.AdamWTable.state8(n, DEV), o.AdamWTable.state8(n, DEV)
    tab = o.AdamWTable([p], [g], [m], [v], exp_avg_scale=[ms], exp_avg_sq_scale=[vs])
    ctr = torch.zeros(1, dtype=torch.int64, device=DEV)
    at = [slice(0, 4096), slice(n // 64 * 32, n // 64 * 32 + 4096), slice((n - 4096) // 32 * 32, n)]
    for t in range(2):
        ctr.fill_(t)
        before = [(_f64(p[s]), m[s].cpu().numpy(), ms[s.start // 32:-(-s.stop // 32)].cpu().numpy(), v[s].cpu().numpy(),
                   vs[s.start // 32:-(-s.stop // 32)].cpu().numpy()) for s in at]
        tab.step(ctr, seed=5, **HYPER)
        for s, (p0, m0, ms0, v0, vs0) in zip(at, before):
            m0, r0, g0 = Q.values8(m0, ms0, True), Q.values8(v0, vs0, False), _f64(g[s])
            rp, rm, rv = Q.adamw(p0, g0, m0, r0 * r0, t + 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
            terms = 0.9 * np.abs(m0) + 0.1 * np.abs(g0)
            upd = HYPER["lr"] / (1 - 0.9 ** (t + 1)) * terms / (np.sqrt(rv) / np.sqrt(1 - 0.999 ** (t + 1)) + 1e-8)
            assert (np.abs(_f64(p[s]) - rp) <= 3 * U * np.abs(p0) + 24 * U * upd).all()
            for x, codes, scales, signed in ((rm, m, ms, True), (np.sqrt(rv), v, vs, False)):
                b = scales[s.start // 32:-(-s.stop // 32)].cpu().numpy()
                got = Q.values8(codes[s].cpu().numpy(), b, signed)
                f = np.repeat(np.exp2(b.astype(np.float64) - 127), 32)[:got.size]
                # within one code of the value: the codes' largest step is 32 (16) scales
                assert (np.abs(got - x) <= (32 if signed else 16) * f * (1 + 1e-5)).all()


def test_adamw_step_as_the_tables_grow():
    """The same tensor in a table of its own and as the first of a table of 40 M elements: the same result."""
    o = _opt()
    n, gen = 5000, torch.Generator().manual_seed(3)
    p0, g0 = torch.randn(n, generator=gen), torch.randn(n, generator=gen) * 1e-2
    got = []
    for more in (0, 40_000_000):
        ps, gs = [p0.to(DEV)], [g0.to(DEV)]
        if more:
            ps.append(torch.zeros(more, device=DEV)), gs.append(torch.ones(more, device=DEV))
        st = [o.AdamWTable.state8(t.numel(), DEV) for t in ps for _ in (0, 1)]
        tab = o.AdamWTable(ps, gs, [s[0] for s in st[::2]], [s[0] for s in st[1::2]], [s[1] for s in st[::2]],
                           [s[1] for s in st[1::2]])
        for t in range(3):
            tab.step(torch.full((1,), t, dtype=torch.int64, device=DEV), seed=9, **HYPER)
        got.append([ps[0], *st[0], *st[1]])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def _eager_and_torch(ps):
    o = _opt()
    mine, ref = [torch.nn.Parameter(p.to(DEV)) for p in ps], [torch.nn.Parameter(p.double()) for p in ps]
    return mine, ref, o.AdamW(mine, lr=0.02, weight_decay=0.1), torch.optim.AdamW(ref, lr=0.02, weight_decay=0.1)


def _close_after(mine, ref, T):
    # as in test_optimizer_matches_torch_adamw
    for x, y in zip(mine, ref):
        tol = T * (4 * U * (y.detach().abs() + 0.02 * T * 4) + 200 * U * 0.02 * 7)
        assert ((x.detach().cpu().double() - y.detach()).abs() <= tol).all()


def test_optimizer_graph_outlives_other_gradients():
    """A captured step goes on with its own gradients' storage while eager steps use another, on one count."""
    gen = torch.Generator().manual_seed(31)
    mine, ref, a, b = _eager_and_torch([torch.randn(50, 20, generator=gen), torch.randn(77, generator=gen)])

    def grads():
        return [torch.randn(p.shape, generator=gen) for p in ref]

    def torch_step(gs):
        for y, g in zip(ref, gs):
            y.grad = g.double()
        b.step()

    gs = grads()
    for x, g in zip(mine, gs):
        x.grad = g.to(DEV)
    a.step()
    torch_step(gs)
    held = [x.grad for x in mine]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        a.step()
    T = 1
    for t in range(4):
        gs = grads()
        for h, g in zip(held, gs):
            h.copy_(g)
        graph.replay()
        torch_step(gs)
        gs = grads()
        for x, g in zip(mine, gs):
            x.grad = g.to(DEV)
        a.step()
        torch_step(gs)
        T += 2
    torch.cuda.synchronize()
    _close_after(mine, ref, T)
    assert float(a.state_dict()["state"][0]["step"]) == T


def test_optimizer_refuses_params_of_different_age():
    gen = torch.Generator().manual_seed(32)
    mine, _, a, _ = _eager_and_torch([torch.randn(5, generator=gen), torch.randn(6, generator=gen)])
    for x in mine:
        x.grad = torch.ones_like(x)
    a.step()
    g1 = mine[1].grad
    mine[1].grad = None
    a.step()
    before = [x.detach().clone() for x in mine]
    mine[1].grad = g1
    with pytest.raises(RuntimeError, match="same number of steps"):
        a.step()
    assert all(torch.equal(x, y) for x, y in zip(mine, before))
    sd = a.state_dict()["state"]
    assert float(sd[0]["step"]) == 2 and float(sd[1]["step"]) == 1


def test_two_tables_on_two_streams():
    """Steps of two tables at once give what they give alone."""
    o = _opt()
    sizes = [(1000, 300), (300,), (257,)]

    def tables():
        out = []
        for seed, bits in ((1, 32), (2, 8)):
            P, G, M, V, MS, VS = _problem(sizes, seed, bits=bits)
            out.append((o.AdamWTable(P, G, M, V, **({} if bits == 32 else dict(exp_avg_scale=MS, exp_avg_sq_scale=VS))), P + M + V))
        return out

    got = []
    for streams in ([torch.cuda.current_stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        tabs = tables()
        ctr = torch.zeros(1, dtype=torch.int64, device=DEV)
        torch.cuda.synchronize()
        for _ in range(20):
            for s, (tab, _) in zip(streams, tabs):
                with torch.cuda.stream(s):
                    tab.step(ctr, seed=3, **HYPER)
        torch.cuda.synchronize()
        got.append([t for _, ts in tabs for t in ts])
    assert all(torch.equal(x, y) for x, y in zip(*got))


def test_adamw_f32_large_tensor():
    """Past 16 M elements: slices of one tensor, its ends among them."""
    o = _opt()
    n = (1 << 24) + 2053
    gen = torch.Generator(device=DEV).manual_seed(13)
    p, m = (torch.randn(n, device=DEV, generator=gen) for _ in "pm")
    g, v = 1e-3 * torch.randn(n, device=DEV, generator=gen), torch.rand(n, device=DEV, generator=gen) * 1e-6
    copy = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    tab = o.AdamWTable([p], [g], [m], [v], copies=[copy])
    at = [slice(0, 4096), slice(n // 2, n // 2 + 4096), slice(n - 4096, n)]
    before = [[_f64(t[s]) for t in (p, g, m, v)] for s in at]
    tab.step(torch.full((1,), 6, dtype=torch.int64, device=DEV), **HYPER)
    for s, (p0, g0, m0, v0) in zip(at, before):
        rp, rm, rv = Q.adamw(p0, g0, m0, v0, 7, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
        terms = 0.9 * np.abs(m0) + 0.1 * np.abs(g0)
        upd = HYPER["lr"] / (1 - 0.9 ** 7) * terms / (np.sqrt(rv) / np.sqrt(1 - 0.999 ** 7) + 1e-8)
        assert (np.abs(_f64(p[s]) - rp) <= 3 * U * np.abs(p0) + 24 * U * upd).all()
        assert (np.abs(_f64(m[s]) - rm) <= 8 * U * terms).all() and (np.abs(_f64(v[s]) - rv) <= 13 * U * rv).all()
    assert torch.equal(copy, p.bfloat16())
