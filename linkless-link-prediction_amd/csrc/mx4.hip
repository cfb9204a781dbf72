// MXFP4: quantisation, its inverse, and the product C = act(A W^T + bias) on the scaled matrix
// instruction (v_mfma_scale_f32_32x32x64_f8f6f4, both operands E2M1 with a power of two per 32 values).
// Format and rounding: include/llp_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "llp_common.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ float as_f32(T x);
template <>
__device__ __forceinline__ float as_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float as_f32<bf16_t>(bf16_t x) { return bf2f(x); }

typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2_any2 __attribute__((ext_vector_type(2), aligned(2)));

// 8 values at any element offset (gfx950's global loads need no alignment), zeros past n
__device__ __forceinline__ void load8(const float* p, int n, float (&x)[8]) {
  if (n >= 8) {
    const f4_any a = *reinterpret_cast<const f4_any*>(p), b = *reinterpret_cast<const f4_any*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? p[i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const bf16_t* p, int n, float (&x)[8]) {
  if (n >= 8) {
    const u4_any2 a = *reinterpret_cast<const u4_any2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? bf2f(p[i]) : 0.f;
  }
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// the scale byte of a block whose largest value has the bits `top`: floor(log2) - 2, at least 2^-127
__device__ __forceinline__ uint32_t mx4_scale(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255u ? 255u : e < 2u ? 0u : e - 2u;
}
// the scale as the f32 that the conversion divides by
__device__ __forceinline__ float mx4_scale_f32(uint32_t s) {
  return __uint_as_float(s ? s << 23 : 0x00400000u);
}
// 8 values to codes: the conversion rounds to nearest even and saturates at 6
__device__ __forceinline__ uint32_t mx4_codes(const float* x, float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
  return c;
}

__device__ __forceinline__ uint32_t quad_umax(uint32_t x) {
  x = umax(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));   // lane ^ 1
  return umax(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));   // lane ^ 2
}

// ---------------------------------------------------------------- quantise
// u / d and u % d for u < 2^31 by a multiplication (Granlund and Montgomery): with 2^(l-1) < d <= 2^l and
// m = ceil(2^(31+l) / d) < 2^32, floor(u / d) = floor(u m / 2^(31+l)).  (A 64-bit division for each 8 values made the
// conversions compute-bound.)
struct FastDiv {
  uint32_t d, m, shift;   // shift = l - 1 of the product's upper word
};
inline FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  if (l == 0) return FastDiv{1, 0, 0};
  return FastDiv{d, (uint32_t)(((1ull << (31 + l)) + d - 1) / d), l - 1};
}
__device__ __forceinline__ uint32_t divided(uint32_t u, const FastDiv& f) {
  return f.m ? __umulhi(u, f.m) >> f.shift : u;
}

// 8 values per lane, a block of 32 per quad: the block's largest by two quad exchanges, 4 bytes of
// codes per lane, one scale byte per quad.  Two such units per thread, 256 apart, both loaded before the first is
// used: 262144 pairs of 235868 rows of 1024 in bf16 196 us, one unit 216, four 227, eight 354.  Bound by memory: 4 or 2 B
// read, 17/32 B written per value: 235868 rows of 1024 in bf16 101 us, 6.1 TB/s (a large copy reaches 4.8).
constexpr int QUANTIZE_UNITS = 2;
template <typename T, bool PAIRS>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(uint32_t units, int K, FastDiv per_row, llp_operand X,
                                                           llp_mx4 out) {
  constexpr int U = QUANTIZE_UNITS;
  const uint32_t u0 = blockIdx.x * (256u * U) + threadIdx.x;
  float x[U][8], y[U][8];
  uint32_t row[U];
  int col[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = u0 + 256 * i < units ? u0 + 256 * i : units - 1;
    row[i] = divided(u, per_row);
    col[i] = (int)(u - row[i] * per_row.d) * 8;
    const int n = K - col[i] < 8 ? (K - col[i] < 0 ? 0 : K - col[i]) : 8;
    load8((const T*)X.ptr + (X.idx ? (int64_t)X.idx[row[i]] : (int64_t)row[i]) * X.ld + col[i], n, x[i]);
    if constexpr (PAIRS)
      load8((const T*)X.ptr2 + (X.idx2 ? (int64_t)X.idx2[row[i]] : (int64_t)row[i]) * X.ld2 + col[i], n, y[i]);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (u0 + 256 * i >= units) break;   // (whole quads: units is a multiple of 16)
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (PAIRS) x[i][j] *= y[i][j];
      top = umax(top, abs_bits(x[i][j]));
    }
    const uint32_t s = mx4_scale(quad_umax(top));
    const uint32_t codes = s == 255u ? 0u : mx4_codes(x[i], mx4_scale_f32(s));
    *(uint32_t*)((uint8_t*)out.codes + (int64_t)row[i] * out.ld_codes + (col[i] >> 1)) = codes;
    if ((threadIdx.x & 3) == 0) ((uint8_t*)out.scales)[(int64_t)row[i] * out.ld_scales + (col[i] >> 5)] = (uint8_t)s;
  }
}

template <bool ONCE, typename V>
__device__ __forceinline__ void store_as(void* p, V v) {   // ONCE: nontemporal, past the caches
  if constexpr (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = v;
}

// the value of code c (E2M1 has f32's fields but for the bias: 2 exponent bits, 1 mantissa bit)
__device__ __forceinline__ float mx4_value(uint32_t c, float scale) {
  const float m = __uint_as_float((c & 7u) << 22) * 0x1p126f;
  return __uint_as_float(__float_as_uint(m) | ((c & 8u) << 28)) * scale;
}

// 16 bytes of a row per lane and unit, so that a store covers whole lines: 8 bf16 or 4 f32 values; two units a thread.
// 262144 x 1024 to bf16: 93 us, 7.3 TB/s (a fill reaches 6.8).
constexpr int DEQUANTIZE_UNITS = 2;
template <typename T, bool ONCE>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(uint32_t units, int K, FastDiv per_row, llp_mx4 X,
                                                             T* __restrict__ Y, int64_t ldy) {
  constexpr int U = DEQUANTIZE_UNITS, V = 16 / sizeof(T);
  const uint32_t u0 = blockIdx.x * (256u * U) + threadIdx.x;
  uint32_t row[U], codes[U], s[U];
  int col[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = u0 + 256 * i < units ? u0 + 256 * i : units - 1;
    row[i] = divided(u, per_row);
    col[i] = (int)(u - row[i] * per_row.d) * V;
    const uint8_t* c = (const uint8_t*)X.codes + (int64_t)row[i] * X.ld_codes + (col[i] >> 1);
    if constexpr (V == 8) codes[i] = *(const uint32_t*)c;
    else codes[i] = *(const uint16_t*)c;
    s[i] = ((const uint8_t*)X.scales)[(int64_t)row[i] * X.ld_scales + (col[i] >> 5)];
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (u0 + 256 * i >= units) break;
    const int n = K - col[i];
    const float f = s[i] == 255u ? __uint_as_float(0x7FC00000u) : mx4_scale_f32(s[i]);
    T* y = Y + (int64_t)row[i] * ldy + col[i];
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = mx4_value(codes[i] >> (4 * j), f);
    if (n >= V) {
      if constexpr (V == 4) {
        store_as<ONCE>(y, f4_any{v[0], v[1], v[2], v[3]});
      } else {
        u4_any2 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = bf16_pair(v[2 * j], v[2 * j + 1]);
        store_as<ONCE>(y, o);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < n) {
          if constexpr (V == 4) y[j] = v[j];
          else y[j] = f2bf(v[j]);
        }
    }
  }
}

// ---------------------------------------------------------------- product
// The matrix instruction's first operand is W and its second A, so that a lane's results lie along a row of C.
// v_mfma_scale_f32_32x32x64: operand lane l holds row l % 32 and the 32 values of block l / 32 of 64 in 4
// registers (16 consecutive bytes of codes), with that block's scale byte; result lane l row l % 32 of C at
// the 16 columns 8 (i / 4) + 4 (l / 32) + i % 4: runs of 4.
struct Mx4Args {
  int64_t M, N, K, Kp, Np;   // Kp, Np: K and N up to 128
  const void* A;         // f32 / bf16 rows
  int64_t lda;
  llp_mx4 A4, W, C4;
  void* C;
  int64_t ldc;
  const float* bias;
  int relu;
  bool streamed;   // whole lines of C past the caches
};

// 8 bf16 of C
__device__ __forceinline__ void store_c8(const Mx4Args& g, int64_t m, int64_t n, const u4v& v) {
  u4_any2* const at = reinterpret_cast<u4_any2*>((bf16_t*)g.C + m * g.ldc + n);
  const u4_any2 c = {v[0], v[1], v[2], v[3]};
  if (g.streamed) __builtin_nontemporal_store(c, at);
  else *at = c;
}

// 32 rows x 64 columns of an f32 C (two tiles of a wave's result) through 8 KB of LDS that the wave has to itself, so that a
// store covers 256 bytes of a row.  Chunk c (16 bytes) of row r at place c ^ r.
__device__ __forceinline__ void store_f32_pair(const Mx4Args& g, uint8_t* part, const float (&y)[2][16], int64_t m0,
                                               int64_t n0, int lane) {
  const int h = lane >> 5, li = lane & 31;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4_t*>(part + li * 256 + (((2 * c + h) ^ (li & 15)) << 4)) =
        float4_t{y[c >> 2][4 * (c & 3)], y[c >> 2][4 * (c & 3) + 1], y[c >> 2][4 * (c & 3) + 2], y[c >> 2][4 * (c & 3) + 3]};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 4), q = lane & 15;
    const float4_t v = *reinterpret_cast<const float4_t*>(part + r * 256 + ((q ^ (r & 15)) << 4));
    f4_any* const at = reinterpret_cast<f4_any*>((float*)g.C + (m0 + r) * g.ldc + n0 + 4 * q);
    const f4_any c = {v[0], v[1], v[2], v[3]};
    if (g.streamed) __builtin_nontemporal_store(c, at);
    else *at = c;
  }
}

// bias of a lane's 16 columns n0 + 8 j + 4 h + i (zero past N)
__device__ __forceinline__ void tile_bias(const Mx4Args& g, int64_t n0, int h, bool full, float (&b)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t n = n0 + 8 * j + 4 * h;
    f4_any v = {0.f, 0.f, 0.f, 0.f};
    if (g.bias) {
      if (full || n + 4 <= g.N) {
        v = *reinterpret_cast<const f4_any*>(g.bias + n);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = n + i < g.N ? g.bias[n + i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) b[4 * j + i] = v[i];
  }
}

// bias and ReLU (a NaN stays: IEEE maximum, not the maxNum of fmaxf)
__device__ __forceinline__ float relu_or(float x, float floor) { return __builtin_elementwise_maximum(x, floor); }
__device__ __forceinline__ void tile_act(const float16_t& acc, const float (&b)[16], int relu, float (&y)[16]) {
  const float floor = relu ? 0.f : -__builtin_inff();
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = relu_or(acc[i] + b[i], floor);
}

// the larger of a lane's value and that of lane ^ 32
__device__ __forceinline__ uint32_t halves_max(uint32_t x) {
  const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return umax(p[0], p[1]);
}

// MXFP4 of the 32 columns of a tile's row (16 in lane l, 16 in lane l ^ 32): the scale byte, and in c the
// codes of columns 0 .. 15 in lanes below 32, of 16 .. 31 above
__device__ __forceinline__ void tile_codes(const float (&y)[16], int h, uint32_t (&c)[2], uint32_t& sc) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = umax(top, abs_bits(y[i]));
  sc = mx4_scale(halves_max(top));
  const float q = mx4_scale_f32(sc);
  uint32_t d[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) d[j] = sc == 255u ? 0u : mx4_codes(y + 8 * j, q);
  // d holds the halves 4 h .. 4 h + 3 of each run of 8 columns
  const auto x = __builtin_amdgcn_permlane32_swap(d[0], d[1], false, false);
  c[0] = (x[0] & 0xFFFFu) | (x[1] << 16);
  c[1] = (x[0] >> 16) | (x[1] & 0xFFFF0000u);
}

// One 32 x 32 tile of a wave's result, perhaps past M or N, stored: bias, ReLU, the output's type
template <int OUT>
__device__ __forceinline__ void store_tile(const Mx4Args& g, const float16_t& acc, const float (&b)[16], int64_t m,
                                           int64_t nb, int h) {
  const bool live = m < g.M;
  float y[16];
  tile_act(acc, b, g.relu, y);
  if constexpr (OUT == 2) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (nb + 8 * (i >> 2) + 4 * h + (i & 3) >= g.N) y[i] = 0.f;
    uint32_t c[2], sc;
    tile_codes(y, h, c, sc);
    if (live && nb < g.Np) {
      uint32_t* o = (uint32_t*)((uint8_t*)g.C4.codes + m * g.C4.ld_codes + nb / 2 + 8 * h);
      o[0] = c[0];
      o[1] = c[1];
      if (h == 0) ((uint8_t*)g.C4.scales)[m * g.C4.ld_scales + nb / 32] = (uint8_t)sc;
    }
  } else if constexpr (OUT == 1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {   // 16 columns: 8 of them in each half of the wave after the exchange
      uint32_t p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = bf16_pair(y[8 * j + 2 * i], y[8 * j + 2 * i + 1]);
      const auto x0 = __builtin_amdgcn_permlane32_swap(p[0], p[2], false, false);
      const auto x1 = __builtin_amdgcn_permlane32_swap(p[1], p[3], false, false);
      const int64_t n = nb + 16 * j + 8 * h;
      bf16_t* o = (bf16_t*)g.C + m * g.ldc + n;
      const uint32_t d[4] = {x0[0], x1[0], x0[1], x1[1]};
      if (live && n + 8 <= g.N) {
        *reinterpret_cast<u4_any2*>(o) = u4_any2{d[0], d[1], d[2], d[3]};
      } else if (live) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < g.N) o[i] = (bf16_t)(d[i >> 1] >> (16 * (i & 1)));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = nb + 8 * j + 4 * h;
      float* o = (float*)g.C + m * g.ldc + n;
      if (live && n + 4 <= g.N) {
        *reinterpret_cast<f4_any*>(o) = f4_any{y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]};
      } else if (live) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < g.N) o[i] = y[4 * j + i];
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
// 16 MT rows x 32 columns of C per workgroup, K split over its 8 waves (128 at a time) and joined through LDS in
// wave order.  What counts here is latency: every load of a wave's step is issued before anything is waited for, and for
// K <= 1024 a wave has one step.  On v_mfma_scale_f32_16x16x128: lane l holds row l % 16 and the 32 values of
// block l / 16 of 128, so that f32 / bf16 rows are quantised in the lane that feeds them, without an exchange; the result's
// lane l has row l % 16 of C at columns 4 (l / 16) + i.  (32 x 32 tiles with K over 4 waves in a loop took
// 11.6 us for 1 x 1024 x 1024.)
// SRC 0: A in MXFP4, 1: f32, 2: bf16.  OUT 0: f32, 1: bf16, 2: MXFP4.
template <int SRC>
__device__ __forceinline__ void load_rows(const Mx4Args& g, int64_t row, int64_t kb, bool ok, u4v (&x)[SRC == 1 ? 8 : SRC == 2 ? 4 : 1],
                                          int& s) {
#pragma unroll
  for (int i = 0; i < (SRC == 1 ? 8 : SRC == 2 ? 4 : 1); ++i) x[i] = u4v{0, 0, 0, 0};
  s = 0;
  if (!ok) return;
  if constexpr (SRC == 0) {
    x[0] = *(const u4v*)((const uint8_t*)g.A4.codes + row * g.A4.ld_codes + kb * 16);
    s = ((const uint8_t*)g.A4.scales)[row * g.A4.ld_scales + kb];
  } else {
    constexpr int PER = SRC == 1 ? 4 : 8;   // values in 16 bytes
    using T = typename std::conditional<SRC == 1, float, bf16_t>::type;
    const T* p = (const T*)g.A + row * g.lda + kb * 32;
    const int64_t left = g.K - kb * 32;
    if (left >= 32) {
#pragma unroll
      for (int i = 0; i < 32 / PER; ++i) {
        const u4_any2 v = *reinterpret_cast<const u4_any2*>(p + PER * i);
        x[i] = u4v{v[0], v[1], v[2], v[3]};
      }
    } else if (left > 0) {   // the row's end: whole pieces of 16 bytes, then one by its elements
      const int whole = (int)left / PER;
      u4v tail = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < PER - 1; ++i)
        if (whole * PER + i < left) {
          if constexpr (SRC == 1) tail[i] = __float_as_uint(p[whole * PER + i]);
          else tail[i >> 1] |= (uint32_t)p[whole * PER + i] << (16 * (i & 1));
        }
#pragma unroll
      for (int i = 0; i < 32 / PER; ++i) {
        if (i < whole) {
          const u4_any2 v = *reinterpret_cast<const u4_any2*>(p + PER * i);
          x[i] = u4v{v[0], v[1], v[2], v[3]};
        } else if (i == whole) {
          x[i] = tail;
        }
      }
    }
  }
}
template <int SRC>
__device__ __forceinline__ v8i as_block(const u4v (&x)[SRC == 1 ? 8 : SRC == 2 ? 4 : 1], int& s) {
  if constexpr (SRC == 0) {
    return v8i{(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3], 0, 0, 0, 0};
  } else {
    float y[32];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      y[i] = SRC == 1 ? __uint_as_float(x[i >> 2][i & 3])
                      : __uint_as_float(i & 1 ? x[i >> 3][(i >> 1) & 3] & 0xFFFF0000u : x[i >> 3][(i >> 1) & 3] << 16);
      top = umax(top, abs_bits(y[i]));
    }
    const uint32_t b = mx4_scale(top);
    const float f = mx4_scale_f32(b);
    s = (int)b;
    v8i v = v8i{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = b == 255u ? 0 : (int)mx4_codes(y + 8 * j, f);
    return v;
  }
}

template <int SRC, int OUT, int MT>
__global__ __launch_bounds__(512) void gemm_mx4_rows_kernel(Mx4Args g) {
  __shared__ float4_t part[8][2 * MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, li = lane & 15;
  const int64_t n0 = (int64_t)blockIdx.x * 32, m0 = (int64_t)blockIdx.y * 16 * MT;
  // bias of the tile that this wave stores (t = wave modulo 2 MT: rows t / 2, columns t % 2)
  float4_t bias = {0.f, 0.f, 0.f, 0.f};
  if (g.bias) {
    const int64_t n = n0 + 16 * (wave & 1) + 4 * q;
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = n + i < g.N ? g.bias[n + i] : 0.f;
  }
  float4_t acc[2][MT];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < MT; ++e) acc[c][e] = float4_t{0.f, 0.f, 0.f, 0.f};
  const int nk = (int)(g.Kp / 128);
  constexpr int XR = SRC == 1 ? 8 : SRC == 2 ? 4 : 1;
  struct Step {
    u4v w[2], x[MT][XR];
    int ws[2], xs[MT];
  };
  auto load = [&](int k, Step& t) {
    const int64_t kb = 4 * (int64_t)k + q;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int64_t n = n0 + 16 * c + li;
      t.w[c] = u4v{0, 0, 0, 0};
      t.ws[c] = 0;
      if (n < g.N) {
        t.w[c] = *(const u4v*)((const uint8_t*)g.W.codes + n * g.W.ld_codes + kb * 16);
        t.ws[c] = ((const uint8_t*)g.W.scales)[n * g.W.ld_scales + kb];
      }
    }
#pragma unroll
    for (int e = 0; e < MT; ++e) load_rows<SRC>(g, m0 + 16 * e + li, kb, m0 + 16 * e + li < g.M, t.x[e], t.xs[e]);
  };
  auto compute = [&](Step& t) {
#pragma unroll
    for (int e = 0; e < MT; ++e) {
      const v8i a = as_block<SRC>(t.x[e], t.xs[e]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const v8i b = v8i{(int)t.w[c][0], (int)t.w[c][1], (int)t.w[c][2], (int)t.w[c][3], 0, 0, 0, 0};
        acc[c][e] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc[c][e], 4, 4, 0, t.ws[c], 0, t.xs[e]);
      }
    }
  };
  if constexpr (MT == 1) {   // the next step's loads in flight under this step's work
    Step t[2];
    if (wave < nk) load(wave, t[0]);
    for (int k = wave; k < nk; k += 16) {
      if (k + 8 < nk) load(k + 8, t[1]);
      compute(t[0]);
      if (k + 8 < nk) {
        if (k + 16 < nk) load(k + 16, t[0]);
        compute(t[1]);
      }
    }
  } else {
    for (int k = wave; k < nk; k += 8) {
      Step t;
      load(k, t);
      compute(t);
    }
  }
  const int live = (int)(nk < 8 ? nk : 8);   // waves that had a step
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int e = 0; e < MT; ++e) part[wave][2 * e + c][lane] = acc[c][e];
  __syncthreads();
  if (OUT != 2 && wave >= 2 * MT) return;
  const int t = wave % (2 * MT), c = t & 1, e = t >> 1;   // (in MXFP4 the other waves repeat a tile up to the barrier)
  float4_t y = part[0][t][lane];
  for (int i = 1; i < live; ++i) y += part[i][t][lane];
  const int64_t m = m0 + 16 * e + li, n = n0 + 16 * c + 4 * q;
  const float floor = g.relu ? 0.f : -__builtin_inff();
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = relu_or(y[i] + bias[i], floor);
  if constexpr (OUT == 2) {
    // a block of 32 columns: the 4 lane groups of two waves, whose largest values meet in LDS
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n + i >= g.N) y[i] = 0.f;
      top = umax(top, abs_bits(y[i]));
    }
    top = umax(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = umax(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    __shared__ uint32_t tops[2 * MT][16];
    if (q == 0) tops[t][li] = top;
    __syncthreads();
    const uint32_t sc = mx4_scale(umax(top, tops[t ^ 1][li]));
    const float f = mx4_scale_f32(sc);
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, y[0], y[1], f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, y[2], y[3], f, 1);
    if (m < g.M && wave < 2 * MT) {
      *(uint16_t*)((uint8_t*)g.C4.codes + m * g.C4.ld_codes + n / 2) = sc == 255u ? 0 : (uint16_t)d;
      if (c == 0 && q == 0) ((uint8_t*)g.C4.scales)[m * g.C4.ld_scales + n0 / 32] = (uint8_t)sc;
    }
  } else if (m < g.M) {
    if constexpr (OUT == 0) {
      float* o = (float*)g.C + m * g.ldc + n;
      if (n + 4 <= g.N) *reinterpret_cast<f4_any*>(o) = f4_any{y[0], y[1], y[2], y[3]};
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < g.N) o[i] = y[i];
    } else {
      bf16_t* o = (bf16_t*)g.C + m * g.ldc + n;
      const uint32_t p0 = bf16_pair(y[0], y[1]), p1 = bf16_pair(y[2], y[3]);
      if (n + 4 <= g.N) *reinterpret_cast<u2_any2*>(o) = u2_any2{p0, p1};
      else
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < g.N) o[i] = (bf16_t)((i < 2 ? p0 : p1) >> (16 * (i & 1)));
    }
  }
}

// ---------------------------------------------------------------- the tiled product
// A workgroup of 4 waves (2 x 2) computes 64 MI rows x 64 NI columns of C (64 x 128, 128 x 128 or 128 x 256), a wave 32 MI x
// 32 NI; four, three or two of them share a CU, so that one's loads and stores run under another's products.  128 of K
// at a time (a step) go through LDS: 64 bytes of codes per row of W and A, by LDS-DMA (global_load_lds)
// into one of three stages, two of them in flight while one is read, so one barrier a step.  Chunk c (16
// bytes) of row r lies at place c ^ place(r) of its row, so that the 16 lanes that read LDS together
// (neighbouring rows at one c) touch all 64 banks.  The scale bytes of 4 steps (16 per row) come at once: 4 of them a step
// would touch as many cache lines as the codes do.  They are read into registers at the first of
// the 4 steps, and the next 16 follow into the same LDS once every wave has read.  SHORT: K of at most
// 3 steps, whose rows hold fewer than 16 scale bytes: 4 bytes at a time, all before the first step.
__device__ __forceinline__ int place(int r) { return ((r >> 2) & 1) | ((((r >> 1) ^ (r >> 3)) & 1) << 1); }
template <int MI, int NI>
struct Mx4Stage {
  static constexpr int TM = 64 * MI, TN = 64 * NI, ROWS = TM + TN;
  static constexpr int BYTES = ROWS * 64;
  static constexpr int DATA = ROWS / 64;                        // 16-byte DMA instructions per wave and step
  static constexpr int SCALE_ROWS = ROWS / 4;                   // rows whose scales a wave fetches
  static constexpr int SCALE = (SCALE_ROWS + 63) / 64;          // DMA instructions for them
  static constexpr int LDS = 3 * BYTES + ROWS * 16 + 16;        // (a read of 16 bytes may begin 12 late)
};

// LDS-DMA from inline asm: the kernel counts its own outstanding loads (vmcnt)
__device__ __forceinline__ void dma16(uint32_t voff, const void* base, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma4(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds) : "memory");
}
__device__ __forceinline__ void dma16p(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(lds) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <int MI, int NI, int OUT, bool SHORT>
__global__ __launch_bounds__(256, NI == 2 ? 3 : 2) void gemm_mx4_kernel(Mx4Args g, FastDiv tiles_n, uint32_t tiles) {
  using S = Mx4Stage<MI, NI>;
  __shared__ __align__(16) uint8_t smem[S::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tile = (uint32_t)llp_xcd_block(blockIdx.x, tiles), tile_m = divided(tile, tiles_n);
  const int64_t n0 = (int64_t)(tile - tile_m * tiles_n.d) * S::TN, m0 = (int64_t)tile_m * S::TM;

  // this wave's DMA sources: 16 rows per data instruction (all of W's or all of A's), clamped to the last
  // valid row (what lies past it is not stored)
  uint32_t voff[S::DATA];
  const uint8_t* base[S::DATA];
#pragma unroll
  for (int i = 0; i < S::DATA; ++i) {
    const int r0 = (wave * S::DATA + i) * 16, r = r0 + (lane >> 2);
    const bool isw = r0 < S::TN;
    const int64_t last = isw ? g.N - 1 - n0 : g.M - 1 - m0;
    int64_t row = isw ? r : r - S::TN;
    row = row < last ? row : last;
    voff[i] = (uint32_t)(row * (isw ? g.W.ld_codes : g.A4.ld_codes)) + (((lane & 3) ^ place(r)) << 4);
    base[i] = isw ? (const uint8_t*)g.W.codes + n0 * g.W.ld_codes : (const uint8_t*)g.A4.codes + m0 * g.A4.ld_codes;
  }
  const uint8_t* sp[S::SCALE];
#pragma unroll
  for (int i = 0; i < S::SCALE; ++i) {
    const int r = wave * S::SCALE_ROWS + i * 64 + lane;
    const bool isw = r < S::TN;
    const int64_t last = isw ? g.N - 1 : g.M - 1;
    int64_t row = isw ? n0 + r : m0 + r - S::TN;
    row = row < last ? row : last;
    sp[i] = isw ? (const uint8_t*)g.W.scales + row * g.W.ld_scales : (const uint8_t*)g.A4.scales + row * g.A4.ld_scales;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int nk = (int)(g.Kp / 128);
  constexpr int SC = 3 * S::BYTES;   // the scales' place
  auto issue = [&](int k, int buf) {
    const uint32_t at = lds0 + buf * S::BYTES;
#pragma unroll
    for (int i = 0; i < S::DATA; ++i) dma16(voff[i], base[i] + (int64_t)k * 64, at + (wave * S::DATA + i) * 1024);
  };
  // scale bytes of steps 4 c .. 4 c + 3; the last 16 of the row where fewer are left
  auto issue_scales = [&](int c) {
    if constexpr (SHORT) {
      for (int k = 0; k < nk; ++k)
#pragma unroll
        for (int i = 0; i < S::SCALE; ++i)
          if (S::SCALE_ROWS % 64 == 0 || i * 64 + lane < S::SCALE_ROWS)
            dma4(sp[i] + 4 * k, lds0 + SC + k * S::ROWS * 4 + (wave * S::SCALE_ROWS + i * 64) * 4);
    } else {
      const int at = 16 * c < 4 * nk - 16 ? 16 * c : 4 * nk - 16;
#pragma unroll
      for (int i = 0; i < S::SCALE; ++i)
        if (S::SCALE_ROWS % 64 == 0 || i * 64 + lane < S::SCALE_ROWS)
          dma16p(sp[i] + at, lds0 + SC + (wave * S::SCALE_ROWS + i * 64) * 16);
    }
  };

  const int wn = wave & 1, wm = wave >> 1, h = lane >> 5, li = lane & 31;
  float16_t acc[NI][MI];
#pragma unroll
  for (int f = 0; f < NI; ++f)
#pragma unroll
    for (int e = 0; e < MI; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][e][i] = 0.f;
  const int wrow = wn * 32 * NI + li, arow = S::TN + wm * 32 * MI + li, sw = place(li);

  // a wave's scale words of 4 steps; byte 2 s + h of a word belongs to the lane: shifted to bytes 0 and 2
  uint32_t ws[NI][4], as[MI][4];
  auto read_scales = [&](int c) {
    const int late = SHORT ? 0 : (16 * c < 4 * nk - 16 ? 0 : 16 * c - (4 * nk - 16));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (SHORT && j == 3) break;
      const uint8_t* at = smem + SC + (SHORT ? j * S::ROWS * 4 : 4 * j + late);
      constexpr int P = SHORT ? 4 : 16;
#pragma unroll
      for (int f = 0; f < NI; ++f) ws[f][j] = *(const uint32_t*)(at + (wrow + 32 * f) * P) >> (8 * h);
#pragma unroll
      for (int e = 0; e < MI; ++e) as[e][j] = *(const uint32_t*)(at + (arow + 32 * e) * P) >> (8 * h);
    }
  };
  issue_scales(0);
  issue(0, 0);
  if (nk > 1) issue(1, 1);
  int buf = 0;
  for (int c = 0; 4 * c < nk; ++c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = 4 * c + j;
      if (k < nk) {
        // what was issued in the last step may stay in flight: one stage, after step 1 the scales too
        if (k + 1 == nk) wait_vm<0>();
        else if (!SHORT && j == 2 && 4 * c + 4 < nk) wait_vm<S::DATA + S::SCALE>();
        else wait_vm<S::DATA>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!SHORT && j == 1 && 4 * c + 4 < nk) issue_scales(c + 1);
        if (k + 2 < nk) issue(k + 2, buf == 0 ? 2 : buf - 1);
        if (j == 0) read_scales(c);
        const uint8_t* st = smem + buf * S::BYTES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          v8i w[NI], a[MI];
#pragma unroll
          for (int f = 0; f < NI; ++f) {
            const u4v q = *(const u4v*)(st + (wrow + 32 * f) * 64 + (((2 * s + h) ^ sw) << 4));
            w[f] = v8i{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
          }
#pragma unroll
          for (int e = 0; e < MI; ++e) {
            const u4v q = *(const u4v*)(st + (arow + 32 * e) * 64 + (((2 * s + h) ^ sw) << 4));
            a[e] = v8i{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
          }
#pragma unroll
          for (int f = 0; f < NI; ++f)
#pragma unroll
            for (int e = 0; e < MI; ++e)
              acc[f][e] = s == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[f], a[e], acc[f][e], 4, 4, 0, (int)ws[f][j], 0, (int)as[e][j])
                                 : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[f], a[e], acc[f][e], 4, 4, 2, (int)ws[f][j], 2, (int)as[e][j]);
        }
        buf = buf == 2 ? 0 : buf + 1;
      }
    }
  }

  const bool full = m0 + S::TM <= g.M && n0 + S::TN <= g.N;
  if constexpr (OUT == 0) {
    if (full) {
      static_assert(4 * 8192 <= S::LDS, "C tiles in LDS");
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the last stage was read by all
#pragma unroll
      for (int f = 0; f < NI; f += 2) {
        const int64_t nb = n0 + (wn * NI + f) * 32;
        float b[2][16], y[2][16];
        tile_bias(g, nb, h, true, b[0]);
        tile_bias(g, nb + 32, h, true, b[1]);
#pragma unroll
        for (int e = 0; e < MI; ++e) {
          tile_act(acc[f][e], b[0], g.relu, y[0]);
          tile_act(acc[f + 1][e], b[1], g.relu, y[1]);
          store_f32_pair(g, smem + wave * 8192, y, m0 + (wm * MI + e) * 32, nb, lane);
        }
      }
      return;
    }
  } else {
    // Through LDS, so that a store covers whole lines of the output's rows (the registers hold runs of 8 bytes,
    // or 2 of codes, in 32 rows).  A wave writes and reads its own part.
    if (full) {
      constexpr int BYTES = OUT == 1 ? 64 * NI : 16 * NI, ROW = BYTES + 16;   // 4 banks on from row to row
      constexpr int PART = 32 * MI * (ROW + (OUT == 2 ? NI : 0));
      static_assert(4 * PART <= S::LDS, "C tile in LDS");
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the last stage was read by all
      uint8_t* part = smem + wave * PART;
#pragma unroll
      for (int f = 0; f < NI; ++f) {
        const int64_t nb = n0 + (wn * NI + f) * 32;
        float b[16];
        tile_bias(g, nb, h, true, b);
#pragma unroll
        for (int e = 0; e < MI; ++e) {
          float y[16];
          tile_act(acc[f][e], b, g.relu, y);
          uint8_t* at = part + (32 * e + li) * ROW;
          if constexpr (OUT == 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint2 p;
              p.x = bf16_pair(y[4 * j], y[4 * j + 1]);
              p.y = bf16_pair(y[4 * j + 2], y[4 * j + 3]);
              *reinterpret_cast<uint2*>(at + 64 * f + 16 * j + 8 * h) = p;
            }
          } else {
            uint32_t c[2], sc;
            tile_codes(y, h, c, sc);
            *reinterpret_cast<uint2*>(at + 16 * f + 8 * h) = make_uint2(c[0], c[1]);
            if (h == 0) part[32 * MI * ROW + (32 * e + li) * NI + f] = (uint8_t)sc;
          }
        }
      }
      constexpr int LANES = BYTES / 16;       // lanes to a row
#pragma unroll
      for (int i = 0; i < 32 * MI * LANES / 64; ++i) {
        const int r = i * (64 / LANES) + lane / LANES, q = lane % LANES;
        const u4v v = *reinterpret_cast<const u4v*>(part + r * ROW + 16 * q);
        const int64_t m = m0 + wm * 32 * MI + r;
        if constexpr (OUT == 1)
          store_c8(g, m, n0 + wn * 32 * NI + 8 * q, v);
        else
          *reinterpret_cast<u4v*>((uint8_t*)g.C4.codes + m * g.C4.ld_codes + (n0 + wn * 32 * NI) / 2 + 16 * q) = v;
      }
      if constexpr (OUT == 2) {
        using Scales = typename std::conditional<NI == 4, uint32_t, uint16_t>::type;   // a row's NI bytes
        static_assert(sizeof(Scales) == NI, "a row's scales as one word");
        for (int r = lane; r < 32 * MI; r += 64)
          *(Scales*)((uint8_t*)g.C4.scales + (m0 + wm * 32 * MI + r) * g.C4.ld_scales + n0 / 32 + wn * NI) =
              *(const Scales*)(part + 32 * MI * ROW + r * NI);
      }
      return;
    }
  }
#pragma unroll
  for (int f = 0; f < NI; ++f) {
    const int64_t nb = n0 + (wn * NI + f) * 32;
    float b[16];
    tile_bias(g, nb, h, false, b);
#pragma unroll
    for (int e = 0; e < MI; ++e) store_tile<OUT>(g, acc[f][e], b, m0 + (wm * MI + e) * 32 + li, nb, h);
  }
}

template <int MI, int NI>
int launch_tiled(const Mx4Args& g, int out, int64_t n_out, hipStream_t s) {
  using S = Mx4Stage<MI, NI>;
  const int64_t tn = (n_out + S::TN - 1) / S::TN, tiles = tn * ((g.M + S::TM - 1) / S::TM);
  LLP_CHECK_ARG(tiles < (1ll << 31), "llp_gemm_nt_mx4: C has too many tiles");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(256), 0, s, g, fast_div((uint32_t)tn), (uint32_t)tiles);
  };
  if (g.Kp <= 384) {
    if constexpr (NI == 4) go(gemm_mx4_kernel<MI, NI, 1, true>);   // (128 x 256 on a short K: bf16 only)
    else out == 0 ? go(gemm_mx4_kernel<MI, NI, 0, true>) : out == 1 ? go(gemm_mx4_kernel<MI, NI, 1, true>) : go(gemm_mx4_kernel<MI, NI, 2, true>);
  } else {
    out == 0 ? go(gemm_mx4_kernel<MI, NI, 0, false>) : out == 1 ? go(gemm_mx4_kernel<MI, NI, 1, false>) : go(gemm_mx4_kernel<MI, NI, 2, false>);
  }
  LLP_LAUNCH_CHECK();
  return LLP_OK;
}

// ---------------------------------------------------------------- the wide product
// What bounds the tiled kernel on long K is the number of its requests to L2: 64 bytes each, 480 a step for
// 128 x 256 columns (126 M for 65536 x 8192 x 2048, 78 % of what the L2 channels take in its time, the matrix
// units at 42 %).  Here a step is 256 of K, so that a row's codes are a whole line of 128 bytes, and a tile 256 x 256,
// a third of the requests.  One workgroup of 8 waves (4 x 2: 64 rows x 128 columns each) per CU takes tile after
// tile; the steps of all its tiles are one sequence, the codes of the next step (the next tile's first) arriving in one
// half of LDS while the other is read.  Row r's chunk c lies at place c ^ place8(r) of its 128 bytes.  K a
// multiple of 256, at least 512.
struct Mx4Wide {
  static constexpr int T = 256, STAGE = 2 * T * 128, SC = 2 * STAGE, BIAS = SC + 2 * T * 16, LDS = BIAS + 2 * 4 * T;
};
static_assert(Mx4Wide::LDS <= 163840, "LDS of a CU");
__device__ __forceinline__ int place8(int r) { return (r >> 1) & 7; }

template <int OUT>
__global__ __launch_bounds__(512, 2) void gemm_mx4_wide_kernel(Mx4Args g, FastDiv tiles_n, uint32_t tiles) {
  using S = Mx4Wide;
  __shared__ __align__(16) uint8_t smem[S::LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, li = lane & 31;
  const int ns = (int)(g.Kp / 256), row_scales = (int)(g.Kp / 32);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  // tiles are dealt in turns of gridDim.x; within a turn each XCD has a contiguous range of them
  uint32_t tile = (uint32_t)llp_xcd_block(blockIdx.x, gridDim.x);
  if (tile >= tiles) return;
  auto tile_m = [&](uint32_t t) { return (int64_t)divided(t, tiles_n) * S::T; };
  auto tile_n = [&](uint32_t t) { return (int64_t)(t - divided(t, tiles_n) * tiles_n.d) * S::T; };

  // DMA sources of the tile that is being fetched: waves 0 .. 3 W's rows, 4 .. 7 A's, 64 each, 8 rows of 128 bytes an
  // instruction; rows past the last valid one repeat it
  const bool isw = wave < 4;
  const uint8_t* const codes = (const uint8_t*)(isw ? g.W.codes : g.A4.codes);
  const uint8_t* const scales = (const uint8_t*)(isw ? g.W.scales : g.A4.scales);
  const int64_t ldc = isw ? g.W.ld_codes : g.A4.ld_codes, lds = isw ? g.W.ld_scales : g.A4.ld_scales;
  const uint32_t ld32 = (uint32_t)ldc;
  const int r8 = (wave & 3) * 64 + (lane >> 3);
  const uint32_t chunk = ((lane & 7) ^ (r8 >> 1 & 3)) << 4;      // (bit 3 of the row: per instruction below)
  int last = 0;
  const uint8_t *base = nullptr, *sp = nullptr;
  const float* bp = nullptr;
  auto aim = [&](uint32_t t) {
    const int64_t r0 = isw ? tile_n(t) : tile_m(t), left = (isw ? g.N : g.M) - 1 - r0;
    last = __builtin_amdgcn_readfirstlane((int)(left < S::T ? left : S::T));
    const int r = (wave & 3) * 64 + lane;
    base = codes + r0 * ldc;
    sp = scales + (r0 + (r < last ? r : last)) * lds;
    bp = isw && g.bias ? g.bias + r0 + (r < last ? r : last) : nullptr;
  };
  // the tile's 256 bias values, in one of two places in turn
  auto issue_bias = [&](uint32_t of) {
    if (isw && g.bias) dma4(bp, lds0 + S::BIAS + (int)(of & 1) * 4 * S::T + wave * 256);
  };
  auto issue = [&](int k, int buf) {
    const uint32_t at = lds0 + buf * S::STAGE + wave * 8192;
    const uint64_t from = (uint64_t)(base + (int64_t)k * 128);
    const uint64_t s = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(from >> 32)) << 32) |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)from);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = r8 + 8 * i;
      dma16((uint32_t)(r < last ? r : last) * ld32 + (chunk ^ ((i & 1) << 6)), (const void*)s, at + i * 1024);
    }
  };
  auto scale_at = [&](int k) { return 8 * k < row_scales - 16 ? 8 * k : row_scales - 16; };   // bytes of steps k, k + 1
  auto issue_scales = [&](int k) { dma16p(sp + scale_at(k), lds0 + S::SC + wave * 1024); };

  const int wn = wave & 1, wm = wave >> 1;
  const int wrow = wn * 128 + li, arow = S::T + wm * 64 + li, sw = place8(li);
  if (!g.bias) *(float*)(smem + S::BIAS + 4 * threadIdx.x) = 0.f;
  aim(tile);
  issue_scales(0);
  issue_bias(0);
  issue(0, 0);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  int buf = 0;
  for (uint32_t turn = 1; tile < tiles; ++turn) {
    const uint32_t next = tile + gridDim.x;
    float16_t acc[4][2];
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[f][e][i] = 0.f;
    uint32_t ws[4][4], as[2][4];
    for (int k2 = 0; k2 < ns; k2 += 2) {
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const int k = k2 + odd;
        if (odd && k == ns) break;
        if (!odd) {
          const int late = 8 * k - scale_at(k);   // 8 where the row's last 16 bytes begin a step early
          auto words = [&](int row, uint32_t (&to)[4]) {
            u4v v = *(const u4v*)(smem + S::SC + row * 16);
            v[0] = late ? v[2] : v[0];
            v[1] = late ? v[3] : v[1];
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = v[j] >> (8 * h);
          };
#pragma unroll
          for (int f = 0; f < 4; ++f) words(wrow + 32 * f, ws[f]);
#pragma unroll
          for (int e = 0; e < 2; ++e) words(arow + 32 * e, as[e]);
        }
        if (k + 1 < ns) {
          if (odd) issue_scales(k + 1);
          issue(k + 1, buf ^ 1);
        } else if (next < tiles) {
          if (!odd) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // all have read these scales
          aim(next);
          issue_scales(0);
          issue_bias(turn);
          issue(0, buf ^ 1);
        }
        const uint8_t* st = smem + buf * S::STAGE;
        u4v w[4], a[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) a[e] = *(const u4v*)(st + (arow + 32 * e) * 128 + ((h ^ sw) << 4));
#pragma unroll
        for (int f = 0; f < 4; ++f) w[f] = *(const u4v*)(st + (wrow + 32 * f) * 128 + ((h ^ sw) << 4));
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int p = 2 * odd + (s >> 1);
          u4v anext[2];
          const int at = (((2 * (s + 1) + h) ^ sw) & 7) << 4;
          if (s < 3)
#pragma unroll
            for (int e = 0; e < 2; ++e) anext[e] = *(const u4v*)(st + (arow + 32 * e) * 128 + at);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const v8i wv = v8i{(int)w[f][0], (int)w[f][1], (int)w[f][2], (int)w[f][3], 0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const v8i av = v8i{(int)a[e][0], (int)a[e][1], (int)a[e][2], (int)a[e][3], 0, 0, 0, 0};
              acc[f][e] = (s & 1) == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, acc[f][e], 4, 4, 0, (int)ws[f][p], 0, (int)as[e][p])
                                       : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wv, av, acc[f][e], 4, 4, 2, (int)ws[f][p], 2, (int)as[e][p]);
            }
            if (s < 3) w[f] = *(const u4v*)(st + (wrow + 32 * f) * 128 + at);   // the next step's, in the same registers
            __builtin_amdgcn_sched_barrier(0);
          }
          if (s < 3)
#pragma unroll
            for (int e = 0; e < 2; ++e) a[e] = anext[e];
        }
        buf ^= 1;
        // the next step's codes have arrived and every wave is done with this step's.  After the tile's last step this
        // comes before its stores, so that they drain under the next tile's first step.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      }
    }

    // The half of LDS that was just read takes C on its way out, so that a store covers whole lines of the output's
    // rows: each wave its own 8 KB, which only its own next fetch overwrites.  Chunk c of row r at place c ^ r.
    uint8_t* const out = smem + (buf ^ 1) * S::STAGE + wave * 8192;
    const int64_t nc = tile_n(tile) + wn * 128, mc = tile_m(tile) + wm * 64;
    const bool full = mc + 64 <= g.M && nc + 128 <= g.N;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t m = mc + 32 * e + li;
      uint32_t row_scales4 = 0;
      float y2[2][16];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int64_t nb = nc + 32 * f;
        __builtin_amdgcn_sched_barrier(0);
        float b[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4_t v = *(const float4_t*)(smem + S::BIAS + (int)((turn - 1) & 1) * 4 * S::T + 4 * (wn * 128 + 32 * f + 8 * j + 4 * h));
#pragma unroll
          for (int i = 0; i < 4; ++i) b[4 * j + i] = v[i];
        }
        if (!full) {
          store_tile<OUT>(g, acc[f][e], b, m, nb, h);
          continue;
        }
        if constexpr (OUT == 0) {
          tile_act(acc[f][e], b, g.relu, y2[f & 1]);
          if (f & 1) store_f32_pair(g, out, y2, mc + 32 * e, nb - 32, lane);
          continue;
        }
        float y[16];
        tile_act(acc[f][e], b, g.relu, y);
        if constexpr (OUT == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint2 q;
            q.x = bf16_pair(y[4 * j], y[4 * j + 1]);
            q.y = bf16_pair(y[4 * j + 2], y[4 * j + 3]);
            *reinterpret_cast<uint2*>(out + li * 256 + (((4 * f + j) ^ (li & 15)) << 4) + 8 * h) = q;
          }
        } else {
          uint32_t c[2], sc;
          tile_codes(y, h, c, sc);
          *reinterpret_cast<uint2*>(out + li * 64 + ((f ^ (li >> 2 & 3)) << 4) + 8 * h) = make_uint2(c[0], c[1]);
          row_scales4 |= sc << (8 * f);
        }
      }
      if (OUT != 0 && full) {
        constexpr int LANES = OUT == 1 ? 16 : 4;       // lanes to a row
#pragma unroll
        for (int i = 0; i < 32 * LANES / 64; ++i) {
          const int r = i * (64 / LANES) + lane / LANES, q = lane % LANES;
          const int64_t mr = mc + 32 * e + r;
          if constexpr (OUT == 1) {
            const u4v v = *reinterpret_cast<const u4v*>(out + r * 256 + ((q ^ (r & 15)) << 4));
            store_c8(g, mr, nc + 8 * q, v);
          } else {
            const u4v v = *reinterpret_cast<const u4v*>(out + r * 64 + ((q ^ (r >> 2 & 3)) << 4));
            *reinterpret_cast<u4v*>((uint8_t*)g.C4.codes + mr * g.C4.ld_codes + nc / 2 + 16 * q) = v;
          }
        }
        if constexpr (OUT == 2)
          if (h == 0) *(uint32_t*)((uint8_t*)g.C4.scales + m * g.C4.ld_scales + nc / 32) = row_scales4;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // its own reads of C, before its next fetch into the same place
    tile = next;
  }
}

int launch_wide(const Mx4Args& g, int out, int64_t n_out, hipStream_t s) {
  const int64_t tn = (n_out + 255) / 256, tiles = tn * ((g.M + 255) / 256);
  LLP_CHECK_ARG(tiles < (1ll << 31), "llp_gemm_nt_mx4: C has too many tiles");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(tiles, 256)), dim3(512), 0, s, g, fast_div((uint32_t)tn), (uint32_t)tiles);
  };
  out == 0 ? go(gemm_mx4_wide_kernel<0>) : out == 1 ? go(gemm_mx4_wide_kernel<1>) : go(gemm_mx4_wide_kernel<2>);
  LLP_LAUNCH_CHECK();
  return LLP_OK;
}

int64_t pad128(int64_t k) { return (k + 127) / 128 * 128; }

template <int MT>
int launch_rows(const Mx4Args& g, int src, int out, int64_t n_out, hipStream_t s) {
  // the grid's second dimension ends at 65,535: longer M in slices
  const int64_t slice = (int64_t)65535 * 16 * MT;
  for (int64_t r = 0; r < g.M; r += slice) {
    Mx4Args h = g;
    h.M = std::min(g.M - r, slice);
    if (src == 0) h.A4.codes = (char*)h.A4.codes + r * h.A4.ld_codes, h.A4.scales = (char*)h.A4.scales + r * h.A4.ld_scales;
    else h.A = (const char*)h.A + r * h.lda * (src == 1 ? 4 : 2);
    if (out == 2) h.C4.codes = (char*)h.C4.codes + r * h.C4.ld_codes, h.C4.scales = (char*)h.C4.scales + r * h.C4.ld_scales;
    else h.C = (char*)h.C + r * h.ldc * (out == 0 ? 4 : 2);
    const dim3 grid((unsigned)((n_out + 31) / 32), (unsigned)((h.M + 16 * MT - 1) / (16 * MT)));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(512), 0, s, h); };
    switch (src * 3 + out) {
      case 0: go(gemm_mx4_rows_kernel<0, 0, MT>); break;
      case 1: go(gemm_mx4_rows_kernel<0, 1, MT>); break;
      case 2: go(gemm_mx4_rows_kernel<0, 2, MT>); break;
      case 3: go(gemm_mx4_rows_kernel<1, 0, MT>); break;
      case 4: go(gemm_mx4_rows_kernel<1, 1, MT>); break;
      case 5: go(gemm_mx4_rows_kernel<1, 2, MT>); break;
      case 6: go(gemm_mx4_rows_kernel<2, 0, MT>); break;
      case 7: go(gemm_mx4_rows_kernel<2, 1, MT>); break;
      default: go(gemm_mx4_rows_kernel<2, 2, MT>); break;
    }
    LLP_LAUNCH_CHECK();
  }
  return LLP_OK;
}

const char* bad_mx4(const llp_mx4* x, int64_t rows, int64_t K) {
  if (!x) return "null";
  if (rows > 0 && (!x->codes || !x->scales)) return "null buffer";
  if (x->ld_codes < pad128(K) / 2 || x->ld_codes % 16 || ((uintptr_t)x->codes & 15)) return "codes need rows of Kp / 2 bytes, 16-B aligned";
  if (x->ld_scales < pad128(K) / 32 || x->ld_scales % 4 || ((uintptr_t)x->scales & 3)) return "scales need rows of Kp / 32 bytes, 4-B aligned";
  return nullptr;
}

// A result that the 256 MB of last-level cache cannot hold passes by the caches, which what is read then keeps
// (131072 x 1024 x 1024 to bf16: 108 -> 93 us, 347 -> 342 with a kernel after it that reads C; a C of half the size would be
// read from the cache: 47 -> 49, 166 -> 175; 262144 x 1024 back to bf16: 122 -> 93)
bool streams(int64_t M, int64_t N, int dtype) { return M * N >= 1ll << (dtype == LLP_F32 ? 26 : 27); }

// rows of a launch: fewer than 2^31 units
int64_t slice_rows(int64_t per_row) { return std::max<int64_t>(1, ((1ll << 31) - 1) / per_row); }

int quantize(int dtype, int64_t M, int64_t K, llp_operand X, llp_mx4 out, hipStream_t s) {
  const int64_t per_row = pad128(K) / 8, slice = slice_rows(per_row);
  const int64_t size = dtype == LLP_F32 ? 4 : 2;
  for (int64_t r = 0; r < M; r += slice) {
    const int64_t n = std::min(M - r, slice);
    llp_operand x = X;
    llp_mx4 o = out;
    if (x.idx) x.idx += r;
    else x.ptr = (const char*)x.ptr + r * x.ld * size;
    if (x.ptr2) {
      if (x.idx2) x.idx2 += r;
      else x.ptr2 = (const char*)x.ptr2 + r * x.ld2 * size;
    }
    o.codes = (char*)o.codes + r * o.ld_codes, o.scales = (char*)o.scales + r * o.ld_scales;
    const uint32_t units = (uint32_t)(n * per_row);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((units - 1) / (256u * QUANTIZE_UNITS) + 1), dim3(256), 0, s, units, (int)K, fast_div((uint32_t)per_row), x, o);
    };
    if (dtype == LLP_F32) x.ptr2 ? go(mx4_quantize_kernel<float, true>) : go(mx4_quantize_kernel<float, false>);
    else x.ptr2 ? go(mx4_quantize_kernel<bf16_t, true>) : go(mx4_quantize_kernel<bf16_t, false>);
    LLP_LAUNCH_CHECK();
  }
  return LLP_OK;
}

}  // namespace

extern "C" int llp_mx4_quantize(int dtype, int64_t M, int64_t K, const llp_operand* X, const llp_mx4* out, void* stream) {
  LLP_CHECK_ARG(dtype == LLP_F32 || dtype == LLP_BF16, "llp_mx4_quantize: rows in f32 or bf16");
  LLP_CHECK_ARG(M >= 0 && K >= 1 && K < (1ll << 31) - 128, "llp_mx4_quantize: M >= 0, 1 <= K < 2^31 - 128");
  if (M == 0) return LLP_OK;
  LLP_CHECK_ARG(X && X->ptr, "llp_mx4_quantize: null pointer");
  LLP_CHECK_ARG(!X->rows_dev, "llp_mx4_quantize: no device row count");
  LLP_CHECK_ARG(!X->idx2 || X->ptr2, "llp_mx4_quantize: idx2 without ptr2");
  const char* why = bad_mx4(out, M, K);
  LLP_CHECK_ARG(!why, "llp_mx4_quantize: out: %s", why);
  return quantize(dtype, M, K, *X, *out, (hipStream_t)stream);
}

extern "C" int llp_mx4_dequantize(int64_t M, int64_t K, const llp_mx4* X, int dtype, void* Y, int64_t ldy, void* stream) {
  LLP_CHECK_ARG(dtype == LLP_F32 || dtype == LLP_BF16, "llp_mx4_dequantize: values in f32 or bf16");
  LLP_CHECK_ARG(M >= 0 && K >= 1 && K < (1ll << 31) - 128 && ldy >= K,
                "llp_mx4_dequantize: M >= 0, 1 <= K < 2^31 - 128, ldy >= K");
  if (M == 0) return LLP_OK;
  LLP_CHECK_ARG(Y, "llp_mx4_dequantize: null pointer");
  const char* why = bad_mx4(X, M, K);
  LLP_CHECK_ARG(!why, "llp_mx4_dequantize: X: %s", why);
  const int64_t v = dtype == LLP_F32 ? 4 : 8, per_row = (K + v - 1) / v, slice = slice_rows(per_row);
  const bool once = streams(M, K, dtype);
  for (int64_t r = 0; r < M; r += slice) {
    const int64_t n = std::min(M - r, slice);
    llp_mx4 x = *X;
    x.codes = (char*)x.codes + r * x.ld_codes, x.scales = (char*)x.scales + r * x.ld_scales;
    const uint32_t units = (uint32_t)(n * per_row);
    auto go = [&](auto kernel, auto* y) {
      hipLaunchKernelGGL(kernel, dim3((units - 1) / (256u * DEQUANTIZE_UNITS) + 1), dim3(256), 0, (hipStream_t)stream, units,
                         (int)K, fast_div((uint32_t)per_row), x, y + r * ldy, ldy);
    };
    if (dtype == LLP_F32) once ? go(mx4_dequantize_kernel<float, true>, (float*)Y) : go(mx4_dequantize_kernel<float, false>, (float*)Y);
    else once ? go(mx4_dequantize_kernel<bf16_t, true>, (bf16_t*)Y) : go(mx4_dequantize_kernel<bf16_t, false>, (bf16_t*)Y);
    LLP_LAUNCH_CHECK();
  }
  return LLP_OK;
}

extern "C" int llp_gemm_nt_mx4(int64_t M, int64_t N, int64_t K, int a_dtype, const llp_operand* A, const llp_mx4* A4,
                               const llp_mx4* W, void* C, int64_t ldc, int c_dtype, const llp_mx4* C4,
                               const float* bias, int act, void* stream) {
  LLP_CHECK_ARG(M >= 0 && N >= 0 && K >= 1 && M < (1ll << 31) && N < (1ll << 31) && K < (1ll << 31),
                "llp_gemm_nt_mx4: M, N >= 0, K >= 1, each < 2^31");
  LLP_CHECK_ARG(act == LLP_ACT_NONE || act == LLP_ACT_RELU, "llp_gemm_nt_mx4: act must be NONE or RELU");
  LLP_CHECK_ARG(A || A4, "llp_gemm_nt_mx4: one of A and A4");
  if (M == 0 || N == 0) return LLP_OK;
  LLP_CHECK_ARG((C != nullptr) != (C4 != nullptr), "llp_gemm_nt_mx4: exactly one of C and C4");
  const char* why = bad_mx4(W, N, K);
  LLP_CHECK_ARG(!why, "llp_gemm_nt_mx4: W: %s", why);
  Mx4Args g{};
  g.M = M, g.N = N, g.K = K, g.Kp = pad128(K), g.Np = pad128(N), g.W = *W, g.bias = bias, g.relu = act == LLP_ACT_RELU;
  int src = 0, out = 2;
  if (A4) {
    why = bad_mx4(A4, M, K);
    LLP_CHECK_ARG(!why, "llp_gemm_nt_mx4: A4: %s", why);
    g.A4 = *A4;
  }
  if (A) {
    LLP_CHECK_ARG(a_dtype == LLP_F32 || a_dtype == LLP_BF16, "llp_gemm_nt_mx4: A in f32 or bf16");
    LLP_CHECK_ARG(A->ptr && !A->idx && !A->ptr2 && !A->idx2 && !A->rows_dev, "llp_gemm_nt_mx4: A must be plain rows");
    LLP_CHECK_ARG(M == 1 || A->ld >= K, "llp_gemm_nt_mx4: A's rows overlap");
    g.A = A->ptr, g.lda = A->ld;
    if (!A4) src = a_dtype == LLP_F32 ? 1 : 2;
  }
  if (C4) {
    why = bad_mx4(C4, M, N);
    LLP_CHECK_ARG(!why, "llp_gemm_nt_mx4: C4: %s", why);
    g.C4 = *C4;
  } else {
    LLP_CHECK_ARG(c_dtype == LLP_F32 || c_dtype == LLP_BF16, "llp_gemm_nt_mx4: C in f32 or bf16");
    LLP_CHECK_ARG(M == 1 || ldc >= N, "llp_gemm_nt_mx4: C's rows overlap");
    g.C = C, g.ldc = ldc;
    out = c_dtype == LLP_F32 ? 0 : 1;
    g.streamed = streams(M, N, c_dtype);
  }
  const int64_t n_out = C4 ? g.Np : N;
  hipStream_t s = (hipStream_t)stream;
  if (A && A4) {
    const int rc = quantize(a_dtype, M, K, *A, *A4, s);
    if (rc != LLP_OK) return rc;
  }
  // Which kernel, by the tiles there are (GPU time in us, rows in MXFP4, bf16 out; 32-bit row offsets within a tile):
  //   up to 512 32 x 32 tiles: the rows kernel, K over a workgroup's waves (512 x 1024 x 1024 6.1, tiled 5.8; 768 rows 8.8 / 6.0;
  //     512 x 8415 -> 256 9.8 / 23.8, 4096 rows 35 / 24; 1024 x 512 x 512 4.3 / 4.6, 2048 rows 5.5 / 4.8), 16 rows at a time
  //     while that makes no more than two workgroups a CU (256 x 1024 x 1024 5.7, 64 at a time 6.3; 512 rows 9.7 / 6.3);
  //   more than 256 128 x 256 tiles, and K in whole steps of 256: wide (12288 x 1024 x 1024 15.0, tiled 16.1; 8192 rows 13.5 / 11.8;
  //     262144 x 2048 x 2048 657 / 845);
  //   else tiled, 64 x 128 while that makes one workgroup a CU (two for K <= 2048, where latency counts): 1024 x 2048 x 2048
  //     9.1, 128 x 128 10.2, 4096 rows 21.1 / 18.1; 8192 x 8415 -> 256 26.4 / 29.6, 12288 rows 37.3 / 30.6;
  //   128 x 128 then, and 128 x 256, where it fits the columns, for long K in no whole steps of 256 (262144 x 8500 -> 256 541,
  //     128 x 128 625; 8192 x 4200 -> 1024, 256 tiles, 31.1 / 32.5; 33000 x 8500 -> 256, 258 of them, 90.6 / 84.8; 16384 rows, 128 of
  //     them, 50.5 / 35.9) and for a bf16 C past the caches (235868 x 128 -> 1024 120 / 137; 235868 x 128 -> 256 27.2 / 23.6).
  const bool near = W->ld_codes < (1 << 23) && (!A4 || A4->ld_codes < (1 << 23));
  auto tiles = [&](int64_t rows, int64_t cols) { return (M + rows - 1) / rows * ((n_out + cols - 1) / cols); };
  if (A4 && near && tiles(32, 32) > 512) {
    if (g.Kp >= 512 && g.Kp % 256 == 0 && tiles(128, 256) > 256) return launch_wide(g, out, n_out, s);
    if (tiles(64, 128) <= (g.Kp <= 2048 ? 512 : 256)) return launch_tiled<1, 2>(g, out, n_out, s);
    const bool fits = (n_out + 127) / 128 % 2 == 0;
    if (fits && ((out == 1 && g.streamed) || (g.Kp > 2048 && tiles(128, 256) >= 256))) return launch_tiled<2, 4>(g, out, n_out, s);
    return launch_tiled<2, 2>(g, out, n_out, s);
  }
  return tiles(16, 32) <= 512 ? launch_rows<1>(g, src, out, n_out, s) : launch_rows<4>(g, src, out, n_out, s);
}
