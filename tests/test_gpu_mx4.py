"""MXFP4 quantisation and product (csrc/mx4.hip, llp_mx) against the definition in 64 bits.

Quantisation is exact: the same codes and scales.  The product of two codes and its scales is exact; K of
them are summed in f32, each sum off by at most 2^-23 of what the sums may reach (the matrix
instruction need not round to nearest): K 2^-23 S with S = sum |a w| + |bias|, plus the bias' sum and the
rounding of the result (2^-24, in bf16 2^-8).
"""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as Q

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def mx():
    import llp_mx
    return llp_mx


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _same(q, x):
    """q holds exactly the codes and scales of x (padding included)."""
    code, s = Q.mx4_codes(x)
    got_s = q.scales.cpu().numpy()
    assert np.array_equal(got_s, s)
    packed = q.codes.cpu().numpy()
    got = np.stack([packed & 15, packed >> 4], 2).reshape(code.shape)
    assert np.array_equal(np.where(got == 8, 0, got), np.where(code == 8, 0, code))       # -0 is 0


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 127), (4, 128), (7, 129), (33, 1433), (300, 257),
                                 (1025, 64), (2, 8415)])
def test_quantize_rows(dt, M, K):
    g = torch.Generator().manual_seed(M * 31 + K)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-12, 12, (M, K), generator=g).float())
    x = torch.where(torch.rand(M, K, generator=g) < 0.2, torch.zeros(()), x).to(TYPES[dt])
    q = mx().quantize(x.to(DEV))
    _same(q, _f64(x))
    for t in (torch.float32, torch.bfloat16):
        assert np.array_equal(_f64(mx().dequantize(q, t)), Q.mx4_round(_f64(x)))


def test_quantize_ties_and_borders():
    """Every tie between two codes, both signs, and largest values on either side of a power of two."""
    v = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.9999, 0.2499, 0.2501, 4.9999, 5.0001])
    rows = []
    for top in (4, 4.0001, 5, 6, 7.9999, 3.9999, 7.0):
        for sign in (1, -1):
            r = np.zeros(64)
            r[:v.size] = sign * np.minimum(v, top)
            r[40] = top
            r[32 + 9:32 + 9 + v.size] = sign * np.minimum(v, top) * 2.0 ** 30
            rows.append(r)
    x = torch.tensor(np.array(rows), dtype=torch.float32)
    _same(mx().quantize(x.to(DEV)), x.double().numpy())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_quantize_extremes(dt):
    """The smallest and largest values of the type, subnormals, and blocks that are all zero."""
    f = torch.finfo(TYPES[dt])
    x = torch.zeros(8, 64)
    x[0, :3] = torch.tensor([f.max, -f.max, f.max / 8])
    x[1, :3] = torch.tensor([f.tiny, f.tiny / 2, f.tiny / 4])
    x[2, 40] = f.smallest_subnormal if hasattr(f, "smallest_subnormal") else f.tiny
    x[3, :2] = torch.tensor([2.0 ** -125, 2.0 ** -126])
    x[4, :2] = torch.tensor([2.0 ** -124, 2.0 ** -128])
    x[5, 5] = -1.0
    x = x.to(TYPES[dt])
    q = mx().quantize(x.to(DEV))
    _same(q, _f64(x))
    assert np.array_equal(_f64(mx().dequantize(q)), Q.mx4_round(_f64(x)))


def test_quantize_nan_and_inf():
    x = torch.randn(3, 100, generator=torch.Generator().manual_seed(1))
    x[0, 40], x[1, 0], x[2, 99] = float("nan"), float("inf"), -float("inf")
    q = mx().quantize(x.to(DEV))
    _same(q, x.double().numpy())
    bad = torch.isnan(mx().dequantize(q)).cpu()
    want = torch.zeros(3, 100, dtype=torch.bool)
    want[0, 32:64] = want[1, :32] = want[2, 96:] = True
    assert torch.equal(bad, want)
    y = mx().linear(x.to(DEV), mx().quantize(torch.randn(40, 100).to(DEV)))
    assert torch.isnan(y).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("K", [1, 40, 256, 1024])
def test_quantize_gathered_and_pairs(dt, K):
    """x[idx] and x[i] * x2[j] of strided rows; the product is not rounded before the block's scale."""
    g = torch.Generator().manual_seed(K)
    h = (torch.randn(50, K + 3, generator=g)).to(TYPES[dt]).to(DEV)[:, 1:K + 1]
    i = torch.randint(0, 50, (333,), generator=g, dtype=torch.int32)
    j = torch.randint(0, 50, (333,), generator=g, dtype=torch.int32)
    i[7] = i[8] = j[7]
    _same(mx().quantize(h, i.to(DEV)), _f64(h)[i.long().numpy()])
    a, b = _f64(h)[i.long().numpy()], _f64(h)[j.long().numpy()]
    _same(mx().quantize(h, i.to(DEV), h, j.to(DEV)), (a * b).astype(np.float32).astype(np.float64))
    full = mx().quantize(h, None, h, None)
    _same(full, (_f64(h) ** 2).astype(np.float32).astype(np.float64))


def test_quantize_writes_its_rows_only():
    m = mx()
    codes = torch.full((9, 64), 0xEE, dtype=torch.uint8, device=DEV)
    scales = torch.full((9, 4), 0xEE, dtype=torch.uint8, device=DEV)
    x = torch.randn(5, 100, device=DEV)
    out = m.MX4(codes[2:7], scales[2:7], 100)
    assert m.quantize(x, out=out) is out
    _same(out, _f64(x))
    for t in (codes, scales):
        assert (t[:2] == 0xEE).all() and (t[7:] == 0xEE).all()


def _check_linear(x, xv, w, wv, b, relu, out_dtype, **kw):
    """x (tensor or MX4) with values xv before quantisation; y against the definition."""
    y = mx().linear(x, w, b, relu=relu, out_dtype=out_dtype, **kw)
    ref, size = Q.mx4_linear(xv, wv, None if b is None else _f64(b), relu)
    K = xv.shape[1]
    tol = (K * 2.0 ** -23 + 2.0 ** -23) * size
    if out_dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (np.abs(ref) + tol)
    got = _f64(y)
    assert got.shape == ref.shape
    bad = np.abs(got - ref) > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), np.abs(got - ref).max())
    return y


# rows: single ones, around the tile sizes and each kernel's range; K and N odd and around the tiles
SHAPES = [(1, 16, 8), (1, 1024, 1024), (1, 1433, 257), (2, 33, 1), (3, 128, 33), (16, 300, 130), (31, 64, 32), (32, 129, 64),
          (33, 256, 128), (47, 1433, 257), (64, 8415, 40), (65, 128, 96), (129, 1000, 129), (255, 512, 256), (257, 384, 300),
          (300, 2048, 64), (513, 128, 513), (1030, 257, 1024), (4099, 64, 72), (2050, 129, 513),
          (33000, 128, 40), (1500, 1433, 700), (5000, 600, 257), (3000, 384, 384), (8200, 100, 300),
          (600, 300, 1000), (600, 2300, 2050), (2050, 640, 520), (5000, 256, 1030), (9000, 384, 260), (8200, 2200, 300),
          (8200, 2200, 1024), (8200, 512, 257), (8231, 1024, 129), (8500, 300, 130), (8192, 1500, 96), (8225, 2048, 160)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("src", ["f32", "bf16", "mx4"])
@pytest.mark.parametrize("out", ["f32", "bf16", "mx4"])
def test_linear(M, K, N, src, out):
    g = torch.Generator().manual_seed(M * 7 + K * 3 + N)
    x = torch.randn(M, K, generator=g)
    x = torch.where(torch.rand(M, K, generator=g) < 0.3, torch.zeros(()), x).to(TYPES.get(src, torch.float32)).to(DEV)
    w = mx().quantize((torch.randn(N, K, generator=g) / K ** 0.5).to(DEV))
    wv = Q.mx4_values(w.codes.cpu().numpy(), w.scales.cpu().numpy(), K)
    b = torch.randn(N, generator=g).to(DEV) if (M + N) % 3 else None
    relu = bool(M % 2)
    xin = mx().quantize(x) if src == "mx4" else x
    if out != "mx4":
        _check_linear(xin, _f64(x), w, wv, b, relu, TYPES[out])
        return
    y = _check_linear(xin, _f64(x), w, wv, b, relu, torch.float32)
    q = mx().linear(xin, w, b, relu=relu, out_dtype="mx4")
    assert q.shape == (M, N)
    _same(q, _f64(y))            # the f32 result's codes, the padding zero


@pytest.mark.parametrize("M", [1, 40, 700])
def test_linear_strided_views_and_given_outputs(M):
    """Rows inside wider tensors at odd offsets, in and out; what lies beside the output stays."""
    m = mx()
    K, N = 200, 70
    g = torch.Generator().manual_seed(M)
    for dt in (torch.float32, torch.bfloat16):
        x = torch.randn(M + 2, K + 5, generator=g).to(dt).to(DEV)[1:M + 1, 3:K + 3]
        w = m.quantize((torch.randn(N, K, generator=g) / 14).to(DEV))
        wv = Q.mx4_values(w.codes.cpu().numpy(), w.scales.cpu().numpy(), K)
        for ot in (torch.float32, torch.bfloat16):
            wide = torch.full((M + 2, N + 9), 5.0, dtype=ot, device=DEV)
            out = wide[1:M + 1, 5:N + 5]
            got = m.linear(x, w, out=out)
            assert got is out
            ref, size = Q.mx4_linear(_f64(x), wv)
            tol = (K + 1) * 2.0 ** -23 * size
            tol = tol + (2.0 ** -8 * (np.abs(ref) + tol) if ot == torch.bfloat16 else 0)
            assert (np.abs(_f64(out) - ref) <= tol).all()
            out.fill_(5.0)
            assert (wide == 5.0).all()


def test_linear_leading_dimensions_and_vectors():
    m = mx()
    x = torch.randn(4, 3, 64, device=DEV)
    w = m.quantize(torch.randn(40, 64, device=DEV))
    y = m.linear(x, w)
    assert y.shape == (4, 3, 40)
    assert torch.equal(y.reshape(12, 40), m.linear(x.reshape(12, 64), w))
    assert torch.equal(m.linear(x[1, 2], w), y[1, 2])


def test_linear_same_for_any_number_of_rows():
    """A row's result does not depend on how many rows go with it, within the sums' order; the codes of
    direct and quantised rows are the same."""
    m = mx()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 320, generator=g).to(DEV)
    w = m.quantize(torch.randn(96, 320, generator=g).to(DEV))
    wv = Q.mx4_values(w.codes.cpu().numpy(), w.scales.cpu().numpy(), 320)
    _, size = Q.mx4_linear(_f64(x), wv)
    full = _f64(m.linear(x, w))
    for n in (1, 5, 64, 65, 128, 400):
        assert (np.abs(_f64(m.linear(x[:n], w)) - full[:n]) <= 2 * 321 * 2.0 ** -23 * size[:n]).all()
        assert (np.abs(_f64(m.linear(m.quantize(x[:n]), w, out_dtype=torch.float32)) - full[:n]) <= 2 * 321 * 2.0 ** -23 * size[:n]).all()


def test_linear_nan_stays_in_its_row():
    m = mx()
    x = torch.randn(70, 256, device=DEV)
    x[3, 100] = float("nan")
    w = m.quantize(torch.randn(64, 256, device=DEV))
    for rows in (slice(0, 5), slice(0, 70)):
        y = m.linear(x[rows], w, relu=True)
        bad = torch.isnan(y)
        assert bad[3].all() and not torch.cat([bad[:3], bad[4:]]).any()
    big, wide = torch.randn(9000, 256, device=DEV), m.quantize(torch.randn(320, 256, device=DEV))
    for i in (0, 130, 8999):
        big[i, 200] = float("inf")
    want = torch.zeros(9000, dtype=torch.bool, device=DEV)
    want[[0, 130, 8999]] = True
    for od in (torch.float32, torch.bfloat16, "mx4"):
        y = m.linear(big, wide, torch.ones(320, device=DEV), relu=True, out_dtype=od)
        bad = torch.isnan(m.dequantize(y) if od == "mx4" else y)
        assert torch.equal(bad.all(1), want) and torch.equal(bad.any(1), want)
    q = m.dequantize(m.linear(x, w, out_dtype="mx4"))
    assert torch.isnan(q[3]).all() and torch.isfinite(torch.cat([q[:3], q[4:]])).all()


def test_empty():
    m = mx()
    w = m.quantize(torch.randn(40, 64, device=DEV))
    for x in (torch.empty(0, 64, device=DEV), m.quantize(torch.empty(0, 64, device=DEV))):
        for od in (torch.float32, torch.bfloat16, "mx4"):
            y = m.linear(x, w, torch.zeros(40, device=DEV), out_dtype=od)
            assert tuple(y.shape) == (0, 40)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    assert m.quantize(torch.randn(5, 64, device=DEV), none).rows == 0
    assert m.dequantize(m.quantize(torch.empty(0, 64, device=DEV))).shape == (0, 64)
    w0 = m.quantize(torch.empty(0, 64, device=DEV))
    assert m.linear(torch.randn(3, 64, device=DEV), w0).shape == (3, 0)


def test_chain_replays_in_a_graph():
    """Pairs quantised, two layers in MXFP4, a bf16 result: captured once, every replay as the eager run."""
    m = mx()
    g = torch.Generator().manual_seed(9)
    h = torch.randn(100, 256, generator=g).bfloat16().to(DEV)
    i, j = (torch.randint(0, 100, (700,), generator=g, dtype=torch.int32).to(DEV) for _ in "ab")
    w1, w2 = (m.quantize((torch.randn(256, 256, generator=g) / 16).to(DEV)) for _ in "ab")
    b = torch.randn(256, generator=g).to(DEV)

    def run():
        q = m.linear(m.quantize(h, i, h, j), w1, b, relu=True, out_dtype="mx4")
        return m.linear(q, w2, b, relu=True, out_dtype=torch.bfloat16)

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for k in range(4):
        h.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(got, run()), k


def test_two_streams_at_once():
    m = mx()
    g = torch.Generator().manual_seed(11)
    xs = [torch.randn(3000, 512, generator=g).to(DEV) for _ in "ab"]
    w = m.quantize(torch.randn(512, 512, generator=g).to(DEV))
    want = [m.linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in "ab"]
    got = [None, None]
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k] = m.linear(xs[k], w)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("K,N", [(128, 1024), (512, 1040), (300, 1024)])
def test_linear_large_result(K, N):
    """A bf16 result of 2^27 values and more is stored past the caches: the f32 result, rounded."""
    m = mx()
    g = torch.Generator(device=DEV).manual_seed(K)
    M = (1 << 17) + 37
    q = m.quantize(torch.randn(M, K, generator=g, device=DEV))
    w, b = m.quantize(torch.randn(N, K, generator=g, device=DEV)), torch.randn(N, generator=g, device=DEV)
    y = m.linear(q, w, b, relu=True, out_dtype=torch.float32)
    assert torch.equal(m.linear(q, w, b, relu=True), y.bfloat16())
    rows = torch.tensor([0, 1, M // 2, M - 38, M - 1], device=DEV)
    part = m.MX4(q.codes[rows], q.scales[rows], K)
    xv, wv = _f64(m.dequantize(part)), _f64(m.dequantize(w))
    ref, size = np.maximum(xv @ wv.T + _f64(b), 0), np.abs(xv) @ np.abs(wv).T + np.abs(_f64(b))
    assert (np.abs(_f64(y[rows]) - ref) <= (K + 1) * 2.0 ** -23 * size).all()


def test_offsets_past_32_bits():
    """Rows whose bytes, elements and results lie past 2^31 and 2^32; conversions in more than one launch."""
    m = mx()
    K, M = 1024, (1 << 24) + 5
    g = torch.Generator(device=DEV).manual_seed(0)
    h = torch.randn(1000, K, generator=g, device=DEV).bfloat16()
    idx = torch.randint(0, 1000, (M,), generator=g, device=DEV, dtype=torch.int32)
    q = m.quantize(h, idx)
    x = m.dequantize(q, torch.bfloat16)
    hq = m.dequantize(m.quantize(h), torch.bfloat16)
    at = [0, 1 << 21, (1 << 22) - 1, 1 << 22, (1 << 23) + 7, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, M - 1]
    for i in at:
        assert torch.equal(x[i], hq[idx[i].long()]), i
    lo = 0
    while lo < M:        # and every row, in pieces
        n = min(1 << 21, M - lo)
        assert torch.equal(x[lo:lo + n], hq[idx[lo:lo + n].long()]), lo
        lo += n
    del x
    w = m.quantize(torch.randn(264, K, generator=g, device=DEV))
    hy = m.linear(m.quantize(h), w, out_dtype=torch.float32)
    y = m.linear(q, w)            # 16.8 M x 264 in bf16: 8.9 GB, of codes of 8.6 GB
    size = (hq.float().abs() @ m.dequantize(w).abs().T)
    for i in at:                  # another kernel's sums: the order differs
        r = int(idx[i])
        assert ((y[i].float() - hy[r]).abs() <= 2 * K * 2.0 ** -23 * size[r] + 2.0 ** -8 * (hy[r].abs() + K * 2.0 ** -23 * size[r])).all(), i


def test_given_outputs_that_overlap_are_refused():
    m = mx()
    x = torch.randn(64, 128, device=DEV)
    q, w = m.quantize(x), m.quantize(torch.randn(128, 128, device=DEV))
    with pytest.raises(ValueError, match="overlaps"):
        m.linear(q, w, out=q)
    with pytest.raises(ValueError, match="overlaps"):
        m.linear(x, w, out=x)
    with pytest.raises(ValueError, match="rows of out overlap"):
        m.dequantize(q, out=torch.empty(1, 128, device=DEV).expand(64, 128))
    with pytest.raises(ValueError, match="rows of out overlap"):
        m.linear(x, w, out=torch.empty(1, 128, device=DEV).expand(64, 128))
    before = m.dequantize(q)
    y = m.linear(q, w, out_dtype="mx4")
    assert torch.equal(m.dequantize(q), before) and m.linear(q, w, out=m.MX4.empty(64, 128, DEV)).shape == y.shape


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("K", [1, 7, 33, 130, 1433])
def test_dequantize_into_a_strided_view(dt, K):
    m = mx()
    x = torch.randn(37, K, generator=torch.Generator().manual_seed(K)).to(DEV)
    q = m.quantize(x)
    wide = torch.full((39, K + 5), 7.0, dtype=TYPES[dt], device=DEV)
    out = wide[1:38, 3:3 + K]
    assert m.dequantize(q, out=out) is out
    assert np.array_equal(_f64(out), Q.mx4_round(_f64(x)))
    wide[1:38, 3:3 + K] = 7.0
    assert (wide == 7.0).all()


def test_quantize_repeated_rows():
    """Rows that are one row in memory, and the same index many times."""
    m = mx()
    row = torch.randn(1, 300, device=DEV)
    _same(m.quantize(row.expand(50, 300)), np.repeat(_f64(row), 50, 0))
    h = torch.randn(3, 300, device=DEV)
    _same(m.quantize(h, torch.full((500,), 2, dtype=torch.int32, device=DEV)), np.repeat(_f64(h[2:]), 500, 0))
    with pytest.raises(RuntimeError, match="overlap"):
        m.linear(row.expand(50, 300), m.quantize(torch.randn(8, 300, device=DEV)))


@pytest.mark.parametrize("M,K,N", [(600, 300, 1000), (2050, 640, 520), (9000, 384, 260), (8200, 512, 512), (40, 1024, 2048)])
def test_replays_of_one_graph_beside_eager_calls(M, K, N):
    """Each kernel captured, replayed three times on new rows, with eager calls of another shape between."""
    m = mx()
    g = torch.Generator(device=DEV).manual_seed(M)
    w, b = m.quantize(torch.randn(N, K, generator=g, device=DEV)), torch.randn(N, generator=g, device=DEV)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    m.linear(x, w, b, relu=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m.linear(x, w, b, relu=True)
        q = m.linear(m.quantize(x), w, b, relu=True, out_dtype="mx4")
    for _ in range(3):
        x.copy_(torch.randn(M, K, generator=g, device=DEV))
        graph.replay()
        m.linear(torch.randn(100, K, generator=g, device=DEV), w)
        torch.cuda.synchronize()
        assert torch.equal(y, m.linear(x, w, b, relu=True))
        assert torch.equal(q.codes, m.linear(m.quantize(x), w, b, relu=True, out_dtype="mx4").codes)
