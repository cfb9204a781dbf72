"""MXFP4 products at shapes that reach each kernel of csrc/mx4.hip in each of its forms, and the C entry's own calls.

Checked in 64 bits on the GPU from the operands' values; K products are summed in f32, each sum off by at most 2^-23 of
what the sums may reach: K 2^-23 S with S = sum |a w| + |bias|, plus the bias' sum.  A bf16 result is the f32 one rounded, an
MXFP4 result the f32 one quantised: the same kernel, the same sums.
"""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def mx():
    import llp_mx
    return llp_mx


def _operands(M, K, N, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV)
    x = torch.where(torch.rand(M, K, generator=g, device=DEV) < 0.3, torch.zeros((), device=DEV), x)
    return x, mx().quantize(torch.randn(N, K, generator=g, device=DEV) / K ** 0.5), torch.randn(N, generator=g, device=DEV)


def _check(y, xq, w, b, relu):
    """An f32 result against the definition, 16,384 rows at a time; b: the bias or None."""
    m, K = mx(), w.cols
    wv = m.dequantize(w).double()
    b = torch.zeros(w.rows, device=DEV) if b is None else b
    for lo in range(0, xq.rows, 16384):
        hi = min(lo + 16384, xq.rows)
        xv = m.dequantize(m.MX4(xq.codes[lo:hi], xq.scales[lo:hi], K)).double()
        ref, size = xv @ wv.t() + b.double(), xv.abs() @ wv.abs().t() + b.double().abs()
        ref = ref.clamp(min=0) if relu else ref
        assert ((y[lo:hi].double() - ref).abs() <= (K + 1) * 2.0 ** -23 * size).all(), lo


def _same(q, y):
    want = mx().quantize(y)
    assert q.shape == want.shape and torch.equal(q.scales, want.scales)
    # (a negative value that rounds to 0 keeps its sign in either)
    assert torch.equal(q.codes, want.codes)


# 128 x 256 tiles over a long K that is no whole number of 256s (one step more than a multiple of 4, one less, three scale groups);
# 256 x 256 tiles, several a workgroup, over an odd and an even number of 256s of K, N past whole tiles
@pytest.mark.parametrize("M,K,N", [(33000, 2170, 256), (32800, 2430, 230), (17000, 2180, 500), (33300, 768, 512), (70000, 700, 600),
                                   (40000, 1280, 440), (70001, 1024, 513), (33300, 8415, 257)])
@pytest.mark.parametrize("bias", [True, False])
def test_many_rows(M, K, N, bias):
    m = mx()
    x, w, b = _operands(M, K, N, M + K)
    b, relu = (b, True) if bias else (None, False)
    q = m.quantize(x)
    del x
    y = m.linear(q, w, b, relu=relu, out_dtype=torch.float32)
    _check(y, q, w, b, relu)
    assert torch.equal(m.linear(q, w, b, relu=relu), y.bfloat16())
    _same(m.linear(q, w, b, relu=relu, out_dtype="mx4"), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(4096, 300, 33), (4090, 512, 20), (3000, 97, 40)])
def test_rows_quantised_on_the_way_into_mxfp4(dtype, M, K, N):
    """The padded columns make more tiles than the caller counts: 64 rows a workgroup."""
    m = mx()
    x, w, b = _operands(M, K, N, 5)
    x = x.to(dtype)
    q = m.quantize(x)
    y = m.linear(q, w, b, relu=True, out_dtype=torch.float32)
    _check(y, q, w, b, True)
    got, want = m.dequantize(m.linear(x, w, b, relu=True, out_dtype="mx4")), m.dequantize(m.linear(q, w, b, relu=True, out_dtype="mx4"))
    # (another kernel's sums: a value beside a border may fall to the next code, under 2 scales away)
    size = m.dequantize(q).abs() @ m.dequantize(w).abs().t() + b.abs()
    step = torch.exp2(m.quantize(y).scales.float() - 127).repeat_interleave(32, 1)[:, :N]
    assert ((got - y).abs() <= step * 2 + K * 2.0 ** -22 * size).all() and ((want - y).abs() <= step * 2 + K * 2.0 ** -22 * size).all()


def _entry(M, N, K, x, w, out, code, b=None, relu=0):
    """The C entry with plain rows and no scratch: they are quantised in the lanes that feed them, however many there are."""
    import llp_hip as K_
    op = K_.Operand(x.data_ptr(), None, None, None, x.stride(0), 0, None)
    four = isinstance(out, mx().MX4)
    K_.launch("llp_gemm_nt_mx4", x.device, M, N, K, K_.dtype_code(x.dtype), C.byref(op), None, C.byref(w.c),
              None if four else out.data_ptr(), 0 if four else out.stride(0), code, C.byref(out.c) if four else None,
              None if b is None else b.data_ptr(), relu)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(2000, 300, 600), (700, 1433, 1000), (65535 * 64 + 70, 5, 2)])
def test_plain_rows_of_any_number(dtype, M, K, N):
    """The last shape takes more than 65,535 workgroups of 64 rows: two launches."""
    m = mx()
    x, w, b = _operands(M, K, N, 6)
    x = x.to(dtype)
    y = _entry(M, N, K, x, w, torch.empty(M, N, device=DEV), 0, b, 1)
    _check(y, m.quantize(x), w, b, True)
    assert torch.equal(_entry(M, N, K, x, w, torch.empty(M, N, dtype=torch.bfloat16, device=DEV), 1, b, 1), y.bfloat16())
    _same(_entry(M, N, K, x, w, m.MX4.empty(M, N, DEV), 0, b, 1), y)


def test_weight_rows_far_apart():
    """Rows 8 MB apart: past what the tiled kernels' 32-bit offsets within a tile take."""
    m = mx()
    M, K, N = 9700, 100, 3
    x, w, b = _operands(M, K, N, 7)
    codes = torch.zeros(N, 1 << 23, dtype=torch.uint8, device=DEV)
    codes[:, :64] = w.codes
    far, q = m.MX4(codes[:, :64], w.scales, K), m.quantize(x)
    y = m.linear(q, far, b, out_dtype=torch.float32)
    _check(y, q, w, b, False)
    assert torch.equal(m.linear(q, far, b), y.bfloat16())
    _same(m.linear(q, far, b, out_dtype="mx4"), y)
