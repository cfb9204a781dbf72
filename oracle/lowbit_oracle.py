"""CPU restatement in 64 bits of the low-bit operators: AdamW (f32 and 8-bit moments) and MXFP4.

Written from the formulas, value by value; nothing here is shared with the kernels.
"""
from __future__ import annotations

import numpy as np

from oracle import llp_oracle as O

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def _log2_floor(x):
    """floor(log2 x) for x > 0, exact."""
    return np.frexp(x)[1] - 1


# ---------------------------------------------------------------- MXFP4
def mx4_codes(x):
    """(codes [M, Kp], scales [M, Kp / 32]) of x [M, K] in MXFP4, Kp = K up to 128; a block with a value
    that is not finite has scale 255 and zero codes."""
    x = np.asarray(x, np.float64)
    M, K = x.shape
    Kp = -(-K // 128) * 128
    b = np.zeros((M, Kp))
    b[:, :K] = x
    b = b.reshape(M, Kp // 32, 32)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[..., None], 0, b)
    top = np.abs(b).max(2)
    e = np.where(top > 0, _log2_floor(np.where(top > 0, top, 1)) - 2, -127).clip(-127)
    y = np.abs(b) / np.exp2(e.astype(np.float64))[..., None]
    # nearest of the 8 magnitudes, ties to the even code
    d = np.abs(np.minimum(y, 6)[..., None] - E2M1)
    best = d.min(-1, keepdims=True)
    first = np.argmax(d == best, -1)
    two = (d == best).sum(-1) == 2
    code = np.where(two & (first % 2 == 1), first + 1, first)
    code = code + 8 * (np.signbit(b) & (b != 0))
    s = np.where(top > 0, e + 127, 0)
    return code.reshape(M, Kp).astype(np.uint8), np.where(bad, 255, s).astype(np.uint8)


def mx4_pack(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).astype(np.uint8)


def mx4_values(packed, scales, K):
    code = np.stack([packed & 15, packed >> 4], 2).reshape(packed.shape[0], -1)
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    f = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * np.repeat(f, 32, 1))[:, :K]


def mx4_round(x):
    """x with every value replaced by the one its MXFP4 code stands for."""
    code, s = mx4_codes(x)
    return mx4_values(mx4_pack(code), s, np.asarray(x).shape[1])


def mx4_linear(x, w, bias=None, relu=False):
    """act(Q(x) w^T + bias) in 64 bits and the sum of the products' magnitudes (for error bounds); w the
    values of an MXFP4 matrix."""
    q = mx4_round(x)
    y, size = q @ w.T, np.abs(q) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return (np.where(y < 0, 0, y) if relu else y), size


# ---------------------------------------------------------------- 8-bit moments
def levels8(signed):
    """The magnitudes of the codes, ascending: E4M3 (0 .. 448) or unsigned 4 + 4 bits (0 .. 496)."""
    bits = 3 if signed else 4
    n = np.arange(127 if signed else 256)
    e, f = n >> bits, n & ((1 << bits) - 1)
    return np.where(e > 0, (1 + f / 2.0 ** bits) * np.exp2(e - 7.0), f / 2.0 ** bits * 2.0 ** -6)


def values8(codes, scales, signed):
    """m (signed) or r = sqrt(v) of a tensor's codes [n] and scales [ceil(n / 32)]."""
    n = codes.size
    f = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    f = np.repeat(f, 32)[:n]
    if signed:
        return levels8(True)[np.minimum(codes & 127, 126)] * np.where(codes & 128, -1.0, 1.0) * f
    return levels8(False)[codes] * f


def draws16(n, tensor, t, seed):
    """The 16-bit draw of each of a tensor's n elements in step t."""
    i = np.arange(n)
    w = O.philox_u32(int(seed), 65536 * int(t) + int(tensor), (i >> 3) * 4 + ((i & 7) >> 1))
    return ((w >> (16 * (i & 1)).astype(np.uint32)) & 0xFFFF).astype(np.int64)


def scales8(size, signed):
    """The scale byte of each block of |m| or r."""
    n = size.size
    b = np.zeros(-(-n // 32) * 32)
    b[:n] = size
    b = b.reshape(-1, 32)
    bad = ~np.isfinite(b).all(1)
    top = np.where(bad, 1, b.max(1))
    lead = 448.0 if signed else 496.0
    k = _log2_floor(np.where(top > 0, top, 1)) - 8
    k = np.where(top > lead * np.exp2(k.astype(np.float64)), k + 1, k).clip(-127, 127)
    return np.where(bad, 255, np.where(top > 0, k + 127, 0)).astype(np.uint8)


def round8(x, w, scales, signed):
    """Stochastic rounding of m, or of v held by its root and where positive at least code 1: (codes, how far
    each draw was from turning the other way, as a share of the distance between the codes)."""
    n = x.size
    f = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32)[:n]
    lv = levels8(signed) if signed else levels8(False) ** 2
    y = np.abs(x) / (f if signed else f * f)
    i = np.clip(np.searchsorted(lv, y, side="right") - 1, 0, lv.size - 2)
    share = (y - lv[i]) / (lv[i + 1] - lv[i])
    if not signed:
        w = (w >> 8) | ((w & 255) << 8)
    u = (w + 0.5) / 65536
    code = np.where(u < share, i + 1, i)
    if signed:
        code = code + 128 * (np.signbit(x) & (code > 0))
    else:
        code = np.where(x > 0, np.maximum(code, 1), code)
    return code.astype(np.uint8), np.abs(u - share)


# ---------------------------------------------------------------- AdamW
def adamw(p, g, m, v, t, lr, betas, eps, decay, sumsq=None, max_norm=1.0):
    """(p', m', v') in 64 bits of one tensor's update number t; sumsq: its clip group's."""
    p, g, m, v = (np.asarray(a, np.float64) for a in (p, g, m, v))
    if sumsq is not None:
        g = g * min(1.0, max_norm / (np.sqrt(float(sumsq)) + 1e-6))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    d = np.sqrt(v) / np.sqrt(1 - betas[1] ** t) + eps
    return p * (1 - lr * decay) - lr / (1 - betas[0] ** t) * m / d, m, v
