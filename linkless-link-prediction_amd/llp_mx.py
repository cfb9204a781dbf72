"""MXFP4 (microscaled 4-bit floating point) matrices for serving the student: quantisation, its
inverse and the product, on the hand-written kernels of csrc/mx4.hip.

  q = quantize(x)                        rows of x (f32 / bf16) in 4.25 bits a value
  q = quantize(h, e0, h, e1)             the predictor's input h[e0] * h[e1] (src/models.py:140)
  y = linear(x, w, bias, relu=True)      relu(Q(x) w^T + bias), w = quantize(weight), laid out once;
                                         x in f32 / bf16, or already in MXFP4; y in f32 / bf16 / MXFP4
  x = dequantize(q)                      the values

Each 32 consecutive values of a row share a power of two; a value is a 4-bit code (0, 0.5, 1, 1.5, 2, 3,
4, 6 and a sign) to nearest, ties to even, saturated at 6.  A block with a NaN or an infinity reads as
NaN.  Products are exact and summed in f32.  There is no gradient: under autograd, with an input that
requires one, the calls raise, and with a dual tensor of forward mode.  Replaces nn.Linear + ReLU of MLP / LinkPredictor in evaluation
(src/models.py:45-54,139-150); used by llp_eval with dtype "mxfp4".
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad

import llp_hip as K


def _direct(rows, cols, outs):
    """Whether rows in f32 / bf16 are quantised inside the product (one launch) or first, once, instead of
    once for each 32 columns of the result: while the product has one workgroup (16 rows x 32 columns) a CU, and K
    leaves each of its waves few steps.  GPU time in us, inside / first, bf16 rows: 128 x 1024 -> 1024 5.1 / 6.3, 256 rows
    8.0 / 7.9; 64 x 2048 -> 2048 7.0 / 7.7, 128 rows 11.7 / 10.5; 512 x 512 -> 512 5.8 / 6.0; 47 x 1433 -> 257 in f32
    6.0 / 6.5; 8 x 4096 -> 64 8.7 / 9.1, 16 rows 10.0 / 9.9; 8 x 8415 -> 256 18.5 / 11.5.  (A second launch costs its
    caller about 4 us more.)"""
    groups = -(-rows // 16) * -(-outs // 32)
    return (cols <= 2048 and groups <= (512 if cols <= 512 else 256)) or (rows <= 8 and cols <= 4096 and groups <= 256)


_FLOATS = (torch.float32, torch.bfloat16)


def _pad(k):
    return -(-k // 128) * 128


class MX4:
    """A [rows, cols] matrix in MXFP4: ``codes`` uint8 [rows, pad / 2] (even element in the low half) and
    ``scales`` uint8 [rows, pad / 32] with pad = cols rounded up to 128 (zero codes behind cols)."""
    __slots__ = ("rows", "cols", "device", "c", "_codes", "_scales", "_both")

    def __init__(self, codes, scales, cols):
        for name, t, per in (("codes", codes, 2), ("scales", scales, 32)):
            if t.dtype != torch.uint8 or t.dim() != 2:
                raise TypeError(f"MX4 {name}: a 2-D uint8 tensor")
            if t.shape[1] * per != _pad(cols) or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError(f"MX4 {name}: rows of {_pad(cols) // per} contiguous bytes for {cols} columns")
        if cols < 1 or codes.shape[0] != scales.shape[0] or codes.device != scales.device:
            raise ValueError("MX4: codes and scales of the same rows, on the same device")
        self.rows, self.cols, self.device = codes.shape[0], int(cols), codes.device
        self._codes, self._scales, self._both = codes, scales, None
        p, one = _pad(self.cols), self.rows <= 1       # (the stride of a single row says nothing)
        self.c = K.Mx4(codes.data_ptr(), scales.data_ptr(), p // 2 if one else codes.stride(0),
                       p // 32 if one else scales.stride(0))

    @staticmethod
    def empty(rows, cols, device):
        p = _pad(cols)
        q = object.__new__(MX4)
        # one allocation, codes first; the two views are made when they are asked for
        q._both = torch.empty(rows * (p // 32) * 17, dtype=torch.uint8, device=device)
        q.rows, q.cols, q.device, q._codes, q._scales = rows, cols, q._both.device, None, None
        at = q._both.data_ptr()
        q.c = K.Mx4(at, at + rows * (p // 2), p // 2, p // 32)
        return q

    @property
    def codes(self):
        if self._codes is None:
            p = _pad(self.cols)
            self._codes = self._both[:self.rows * (p // 2)].view(self.rows, p // 2)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            p = _pad(self.cols)
            self._scales = self._both[self.rows * (p // 2):].view(self.rows, p // 32)
        return self._scales

    @property
    def shape(self):
        return (self.rows, self.cols)


def _row_stride(out, what):
    """The row stride of a given 2-D output, whose rows must not share memory."""
    rows, cols = out.shape
    if rows > 1 and out.stride(0) < cols:
        raise ValueError(f"{what}: the rows of out overlap")
    return out.stride(0) if rows > 1 else cols


def _spans(t):
    """Where the rows of a matrix lie: [(first byte, rows, bytes from row to row, bytes of a row)]."""
    rows, cols = t.shape
    if not rows:
        return []
    if isinstance(t, MX4):
        p = _pad(cols)
        at = [(t.c.codes, rows, t.c.ld_codes, p // 2), (t.c.scales, rows, t.c.ld_scales, p // 32)]
    else:
        size = t.element_size()
        at = [(t.data_ptr(), rows, (t.stride(0) if rows > 1 else cols) * size, cols * size)]
    # rows that overlap one another, as an expanded tensor's: one piece
    return [(a, n, s, w) if s >= w else (a, 1, 1, (n - 1) * s + w) for a, n, s, w in at]


def _apart(what, out, *inputs):
    """A given output shares no memory with what the call reads."""
    mine = _spans(out)
    if len(mine) == 2 and K.rows_meet(*mine):
        raise ValueError(f"{what}: out's codes and scales overlap")
    for t in inputs:
        if any(K.rows_meet(a, b) for a in _spans(t) for b in mine):
            raise ValueError(f"{what}: out overlaps an input")


def _on_gpu(dev):
    if dev.type != "cuda":
        raise RuntimeError("LLP ops run only on the MI355X HIP device (got a CPU tensor; no CPU fallback)")


def _no_gradient(t, what):
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what}: MXFP4 has no gradient; call it under torch.no_grad()")
    # (the tangent of a dual tensor, which torch.no_grad() leaves on; outside of every dual level there is none)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{what}: MXFP4 has no gradient, forward mode neither; unpack the dual tensor")


def _rows2d(x, what):
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{what}: a 2-D tensor with contiguous rows")
    if x.dtype not in _FLOATS:
        raise TypeError(f"{what}: f32 or bf16, not {x.dtype}")
    if not x.is_cuda:
        _on_gpu(x.device)
    _no_gradient(x, what)


def _index(i, x, what):
    if i is None:
        return
    if i.dtype != torch.int32 or i.dim() != 1 or not i.is_contiguous():
        raise TypeError(f"{what}: a contiguous 1-D int32 tensor")
    if i.device != x.device:
        raise ValueError(f"{what}: on {i.device}, the rows on {x.device}")


def quantize(x, idx=None, x2=None, idx2=None, out=None):
    """MXFP4 of x[idx] (of x2[idx2] * x[idx], formed in f32, with x2); idx None: all rows.  The indices
    must lie within the rows (they are read on the device and not checked)."""
    _rows2d(x, "quantize")
    _index(idx, x, "quantize idx")
    rows = x.shape[0] if idx is None else idx.shape[0]
    if x2 is None:
        if idx2 is not None:
            raise ValueError("quantize: idx2 without x2")
        op = K.Operand(x.data_ptr(), K.ptr(idx), None, None, x.stride(0), 0, None)
    else:
        _rows2d(x2, "quantize x2")
        _index(idx2, x, "quantize idx2")
        if x2.dtype != x.dtype or x2.device != x.device or x2.shape[1] != x.shape[1]:
            raise ValueError("quantize: x and x2 of one dtype, device and width")
        if (x2.shape[0] if idx2 is None else idx2.shape[0]) != rows:
            raise ValueError("quantize: x[idx] and x2[idx2] differ in rows")
        op = K.Operand(x.data_ptr(), K.ptr(idx), x2.data_ptr(), K.ptr(idx2), x.stride(0), x2.stride(0), None)
    if rows and min(x.shape[0], rows if x2 is None else x2.shape[0]) == 0:
        raise ValueError("quantize: indices into no rows")
    if x.shape[1] < 1:
        raise ValueError("quantize: no columns")
    if out is None:
        out = MX4.empty(rows, x.shape[1], x.device)
    elif out.shape != (rows, x.shape[1]) or out.device != x.device:
        raise ValueError(f"quantize: out is {out.shape} on {out.device}, the rows are {(rows, x.shape[1])} on {x.device}")
    else:
        _apart("quantize", out, x, *(t if t.dim() == 2 else t.view(1, -1) for t in (idx, x2, idx2) if t is not None))
    K.launch("llp_mx4_quantize", x.device, K.dtype_code(x.dtype), rows, x.shape[1], C.byref(op), C.byref(out.c))
    return out


def dequantize(q, dtype=torch.float32, out=None):
    """The values of q (exact in f32; in bf16 too, down to 2^-133)."""
    _on_gpu(q.device)
    if out is None:
        out = torch.empty(q.rows, q.cols, dtype=dtype, device=q.device)
    elif tuple(out.shape) != q.shape or out.device != q.device or (q.cols > 1 and out.stride(1) != 1):
        raise ValueError("dequantize: out needs q's shape, on its device, with contiguous rows")
    else:
        _apart("dequantize", out, q)
    K.launch("llp_mx4_dequantize", q.device, q.rows, q.cols, C.byref(q.c), K.dtype_code(out.dtype), out.data_ptr(),
             _row_stride(out, "dequantize"))
    return out


def linear(x, w, bias=None, relu=False, out_dtype=None, out=None):
    """act(Q(x) w^T + bias): x [..., cols] in f32 / bf16 or an MX4, w an MX4 [N, cols], bias [N].
    out_dtype torch.float32 / torch.bfloat16 / "mx4" (default x's dtype; bf16 for an MX4 x); ``out``: a
    2-D tensor with contiguous rows, or an MX4, written in place of a new one."""
    lead = op = None
    four_in = isinstance(x, MX4)
    if not four_in:
        if x.dim() != 2:
            lead = x.shape[:-1]
            x = x.reshape(-1, x.shape[-1])
        _rows2d(x, "linear")
    else:
        _on_gpu(x.device)
    rows, width = x.shape
    N, dev = w.rows, x.device
    if width != w.cols or dev != w.device:
        raise ValueError(f"linear: x has {width} columns on {dev}, w has {w.cols} on {w.device}")
    if bias is not None:
        _no_gradient(bias, "linear")
        if bias.shape != (N,) or bias.device != dev:
            raise ValueError(f"linear: bias of {N} values on {dev}")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.detach().float().contiguous()
    if out is None:
        if out_dtype is None:
            out_dtype = torch.bfloat16 if four_in else x.dtype
        four_out, ldc = out_dtype == "mx4", N
        out = MX4.empty(rows, N, dev) if four_out else torch.empty((rows, N), dtype=out_dtype, device=dev)
    elif tuple(out.shape) != (rows, N) or out.device != dev or lead is not None:
        raise ValueError(f"linear: out is {tuple(out.shape)} on {out.device}, the result is {(rows, N)} on {dev}")
    else:
        _apart("linear", out, x, w, *([] if bias is None else [bias.view(1, N)]))
        four_out = isinstance(out, MX4)
        if not four_out:
            if N > 1 and out.stride(1) != 1:
                raise TypeError("linear: out in f32 or bf16 with contiguous rows")
            ldc = _row_stride(out, "linear")
    if not four_out and out.dtype not in _FLOATS:
        raise TypeError("linear: out in f32 or bf16 with contiguous rows")
    code, x4 = 0, x if four_in else None
    if not four_in:
        op, code = C.byref(K.Operand(x.data_ptr(), None, None, None, x.stride(0), 0, None)), K.dtype_code(x.dtype)
        if not _direct(rows, width, N):
            x4 = MX4.empty(rows, width, dev)      # scratch: the call quantises x into it first
    c4 = None if x4 is None else C.byref(x4.c)
    act = K.ACT_RELU if relu else K.ACT_NONE
    b = None if bias is None else bias.data_ptr()
    if four_out:
        K.launch("llp_gemm_nt_mx4", dev, rows, N, width, code, op, c4, C.byref(w.c), None, 0, 0,
                 C.byref(out.c), b, act)
        return out
    K.launch("llp_gemm_nt_mx4", dev, rows, N, width, code, op, c4, C.byref(w.c),
             out.data_ptr(), ldc, K.dtype_code(out.dtype), None, b, act)
    return out if lead is None else out.reshape(*lead, N)
