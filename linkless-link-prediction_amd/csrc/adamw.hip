// AdamW over many tensors in one launch, with its moments in f32 or in 8 bits.
//
//   g' = c g (c the clip coefficient of the tensor's group), t = *step + 1
//   m' = b1 m + (1 - b1) g'            v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// 8-bit moments.  Each 32 consecutive elements of a tensor share a power of two 2^k (one byte,
// k + 127; 255 = the block holds a NaN or an infinity): m is kept as E4M3 codes, r = sqrt(v) as unsigned codes of
// 4 exponent and 4 mantissa bits (bias 7, largest 496, no NaN code).  k is the least power that
// holds the block's largest value (448 / 496 times 2^k), so nothing saturates.  The root is what is kept because
// its range is half of v's in exponents: codes of 2^-10 .. 496 are v over 2^38 within a block.
// Rounding is stochastic, from one 16-bit Philox draw per element, and keeps the MEAN of m and of
// v = r^2 (not of r, whose square would grow by the rounding's variance, up to 0.1 % a step, as much as
// its decay of 1 - b2 = 0.1 %).  Rounding to nearest would do worse still: a step changes v by 0.1 %,
// a code is 3 to 6 % wide, and v would never move down.
// One exception: where v' > 0 the code of r is at least 1.  A root rounded to 0 beside a first moment that is not would make the
// next update m' / eps (with gradient sizes log-normal of sigma 2 within a block, 5 % of them at a time, single updates of 230 lr;
// 1.7 lr with the least code, 1.2 lr in f32).  The mean of v below the least code's square grows by less than that square.
// The update of p uses m' and v' before they are rounded.
//
// Bound by memory: per element 8 B of p, 4 (2) of g, and 16 B of f32 moments or 4.1 B of 8-bit ones.  34 M f32
// elements with a bf16 copy, into other buffers: 189 us at 5.4 TB/s with f32 moments; 1e8 in place 548 us (5.5 TB/s), with
// 8-bit moments 338 us (5.3 TB/s; a large copy reaches 4.8).  500,000 elements: a kernel of 5.7 and 6.7 us (rocprofv3; 5.0 and 5.6
// apart in a graph), of which memory would take 2.9 and 1.5: latency, of the chain work item -> descriptor -> data and of the
// step's constants, which every thread computes in f64.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "llp_common.h"

namespace {

// One work item: 2,048 consecutive elements of one tensor, 8 per thread, so that a quad of lanes
// holds a block of 32 and a thread one Philox block (4 words = 8 draws).
constexpr int64_t AW_ITEM = 2048;

// 16 bytes at any address: the global loads and stores of gfx950 need no alignment, so gradients
// that are views of a flat buffer at odd offsets take the same path as aligned tensors.
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2_any1 __attribute__((ext_vector_type(2), aligned(1)));

// ONCE: nontemporal, past the caches
template <bool ONCE, typename V>
__device__ __forceinline__ V load_as(const void* p) {
  if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else return *reinterpret_cast<const V*>(p);
}
template <bool ONCE, typename V>
__device__ __forceinline__ void store_as(void* p, V v) {
  if constexpr (ONCE) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = v;
}

template <bool ONCE>
__device__ __forceinline__ void load8(const float* p, int64_t e, int n, float (&x)[8]) {
  if (n == 8) {
    const f4_any a = load_as<ONCE, f4_any>(p + e), b = load_as<ONCE, f4_any>(p + e + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? p[e + i] : 0.f;
  }
}
template <bool ONCE>
__device__ __forceinline__ void load8(const bf16_t* p, int64_t e, int n, float (&x)[8]) {
  if (n == 8) {
    const u4_any2 a = load_as<ONCE, u4_any2>(p + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(a[i] << 16);
      x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? bf2f(p[e + i]) : 0.f;
  }
}

template <bool ONCE>
__device__ __forceinline__ void store8(float* p, int64_t e, int n, const float (&x)[8]) {
  if (n == 8) {
    store_as<ONCE>(p + e, f4_any{x[0], x[1], x[2], x[3]});
    store_as<ONCE>(p + e + 4, f4_any{x[4], x[5], x[6], x[7]});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[e + i] = x[i];
  }
}
template <bool ONCE>
__device__ __forceinline__ void store8(bf16_t* p, int64_t e, int n, const float (&x)[8]) {
  if (n == 8) {
    u4_any2 a;
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
    store_as<ONCE>(p + e, a);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[e + i] = f2bf(x[i]);
  }
}

__device__ __forceinline__ void load_codes(const uint8_t* p, int64_t e, int n, uint32_t (&w)[2]) {
  if (n == 8) {
    const u2_any1 a = *reinterpret_cast<const u2_any1*>(p + e);
    w[0] = a[0], w[1] = a[1];
  } else {
    w[0] = w[1] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) w[i >> 2] |= (uint32_t)p[e + i] << (8 * (i & 3));
  }
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t e, int n, const uint32_t (&w)[2]) {
  if (n == 8) {
    *reinterpret_cast<u2_any1*>(p + e) = u2_any1{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[e + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
  }
}

// 2^(s - 127), NaN for s = 255
__device__ __forceinline__ float scale_value(uint32_t s) {
  const float f = s ? __uint_as_float(s << 23) : __uint_as_float(0x00400000u);
  return s == 255u ? __uint_as_float(0x7FC00000u) : f;
}

__device__ __forceinline__ void decode_m(const uint32_t (&w)[2], uint32_t s, float (&m)[8]) {
  const float f = scale_value(s);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
    m[4 * i] = a[0] * f, m[4 * i + 1] = a[1] * f, m[4 * i + 2] = b[0] * f, m[4 * i + 3] = b[1] * f;
  }
}
// r = sqrt(v): the code's bits are an f32's exponent and mantissa but for the bias
__device__ __forceinline__ void decode_r(const uint32_t (&w)[2], uint32_t s, float (&r)[8]) {
  const float f = scale_value(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = (w[i >> 2] >> (8 * (i & 3))) & 0xFFu;
    r[i] = (__uint_as_float(c << 19) * 0x1p120f) * f;
  }
}

// the largest of a quad's values as unsigned bits (a NaN or infinity stays on top)
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true);   // lane ^ 1
  x = x > y ? x : y;
  const uint32_t z = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true);   // lane ^ 2
  return x > z ? x : z;
}
// the scale byte of a block whose largest value has the bits `top`; `lead`: the mantissa bits of the
// largest code (1.75 * 2^8 = 448, 1.9375 * 2^8 = 496)
__device__ __forceinline__ uint32_t scale_byte(uint32_t top, uint32_t lead) {
  if (top >= 0x7F800000u) return 255u;
  const int s = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > lead ? 1 : 0);
  return s < 0 ? 0u : (uint32_t)s;
}
// 2^-(s - 127) for s <= 254
__device__ __forceinline__ float scale_inverse(uint32_t s) {
  return s == 254u ? __uint_as_float(0x00400000u) : __uint_as_float((254u - s) << 23);
}

// y (|y| <= 448) to an E4M3 code, up where u < the fraction, u = (w + 1/2) / 65536: the 20 bits below
// the code's mantissa plus (1 - u) carry into it.  Below 2^-6 the codes are 2^-9 apart; adding 2^-6
// gives the value that spacing.
__device__ __forceinline__ uint32_t round_m(float y, uint32_t w) {
  const float a = fabsf(y);
  const bool sub = a < 0x1p-6f;
  const uint32_t t = __float_as_uint(sub ? a + 0x1p-6f : a);
  const uint32_t c = ((t + (((w ^ 0xFFFFu) << 4) | 7u)) >> 20) - (sub ? 968u : 960u);
  return c | ((__float_as_uint(y) >> 24) & 0x80u);
}
// r (y = r 2^-k <= 496, x = v 2^-2k) to a code, up where u < (x - lo^2) / (hi^2 - lo^2), at least `least`
__device__ __forceinline__ uint32_t round_r(float y, float x, uint32_t w, uint32_t least) {
  const bool sub = y < 0x1p-6f;
  const float off = sub ? 0x1p-6f : 0.f;
  const uint32_t t = __float_as_uint(y + off) & 0xFFF80000u;
  const float lo = __uint_as_float(t) - off, hi = __uint_as_float(t + 0x80000u) - off;
  const float den = (hi - lo) * (hi + lo), num = fmaf(-lo, lo, x);
  const float u = fmaf((float)w, 0x1p-16f, 0x1p-17f);
  uint32_t c = (t >> 19) - (sub ? 1936u : 1920u);
  c += u * den < num ? 1u : 0u;
  c = c < least ? least : c;
  return c > 255u ? 255u : c;
}

// the working copy, rows copy_ld apart (0: as the parameter)
template <bool ONCE>
__device__ __forceinline__ void store_copy(const llp_adamw_desc& d, int64_t e, int n, const float (&p)[8]) {
  if (d.copy_ld == 0 || d.copy_ld == d.cols) {
    if (d.copy_dtype == LLP_BF16) store8<ONCE>((bf16_t*)d.copy, e, n, p);
    else store8<ONCE>((float*)d.copy, e, n, p);
    return;
  }
  int64_t c = e % d.cols, at = e / d.cols * d.copy_ld + c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < n) {
      if (d.copy_dtype == LLP_BF16) ((bf16_t*)d.copy)[at] = f2bf(p[i]);
      else ((float*)d.copy)[at] = p[i];
    }
    ++at;
    if (++c == d.cols) c = 0, at += d.copy_ld - d.cols;
  }
}

// beta^t by squaring (t >= 1)
__device__ __forceinline__ double int_pow(double b, int64_t t) {
  double r = 1.0;
  while (t > 0) {
    if (t & 1) r *= b;
    b *= b;
    t >>= 1;
  }
  return r;
}

struct AdamWArgs {
  double lr, beta1, beta2, eps, decay, max_norm;
  uint64_t seed;
};

template <int BITS, bool ONCE, typename P, typename G>
__global__ __launch_bounds__(256) void adamw_kernel(const llp_adamw_desc* __restrict__ descs,
                                                    const int32_t* __restrict__ work, int64_t n_work,
                                                    const float* __restrict__ sumsq, AdamWArgs a,
                                                    const int64_t* __restrict__ step) {
  const int64_t t = *step + 1;
  const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2);
  const float inv_bc2 = (float)(1.0 / sqrt(1.0 - int_pow(a.beta2, t)));
  const float size = (float)(a.lr / (1.0 - int_pow(a.beta1, t)));
  const float keep = (float)(1.0 - a.lr * a.decay), eps = (float)a.eps;
  for (int64_t w = blockIdx.x; w < n_work; w += gridDim.x) {
    const int tensor = work[2 * w];
    const llp_adamw_desc d = descs[tensor];
    const int64_t e = (int64_t)work[2 * w + 1] * AW_ITEM + 8 * threadIdx.x;
    const int n = e >= d.numel ? 0 : (int)(d.numel - e < 8 ? d.numel - e : 8);
    float coef = 1.f;
    if (sumsq) {   // clip_grad_norm_: min(1, max_norm / (norm + 1e-6)), a NaN norm kept
      const float q = (float)a.max_norm / (sqrtf(sumsq[d.group]) + 1e-6f);
      coef = (q != q) ? q : fminf(q, 1.f);
    }
    float g[8], p[8], m[8], v[8], r[8];
    load8<ONCE>((const G*)d.grad, e, n, g);
    load8<ONCE>((const P*)d.param, e, n, p);
    if constexpr (BITS == 32) {
      load8<false>((const float*)d.exp_avg, e, n, m);
      load8<false>((const float*)d.exp_avg_sq, e, n, v);
    } else {
      uint32_t cm[2], cr[2];
      load_codes((const uint8_t*)d.exp_avg, e, n, cm);
      load_codes((const uint8_t*)d.exp_avg_sq, e, n, cr);
      decode_m(cm, n ? d.exp_avg_scale[e >> 5] : 0u, m);
      decode_r(cr, n ? d.exp_avg_sq_scale[e >> 5] : 0u, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r[i] * r[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // (the pragma holds to the end of this block)
      // every product and sum rounded by itself, in the formula's order: the draws then fall as they
      // do for elementary f32 operations
#pragma clang fp contract(off)
      const float gi = g[i] * coef;
      m[i] = b1 * m[i] + c1 * gi;
      v[i] = b2 * v[i] + (c2 * gi) * gi;
      r[i] = sqrtf(v[i]);
      p[i] = p[i] * keep - size * (m[i] / (r[i] * inv_bc2 + eps));
    }
    store8<ONCE>((P*)d.param_out, e, n, p);
    if (d.copy) {
      if constexpr (sizeof(P) == 2)   // an f32 copy of a bf16 param holds the param, as the transposed one does
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = bf2f(f2bf(p[i]));
      store_copy<ONCE>(d, e, n, p);
    }
    if constexpr (BITS == 32) {
      store8<false>((float*)d.exp_avg_out, e, n, m);
      store8<false>((float*)d.exp_avg_sq_out, e, n, v);
    } else {
      uint32_t tm = 0, tr = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= n) m[i] = v[i] = r[i] = 0.f;
        const uint32_t am = __float_as_uint(m[i]) & 0x7FFFFFFFu, ar = __float_as_uint(r[i]) & 0x7FFFFFFFu;
        tm = tm > am ? tm : am;
        tr = tr > ar ? tr : ar;
      }
      const uint32_t sm = scale_byte(quad_max(tm), 0x600000u), sr = scale_byte(quad_max(tr), 0x780000u);
      const uint4 draw = philox4((uint64_t)(e >> 3), (uint64_t)t * 65536u + (uint64_t)tensor, a.seed);
      uint32_t cm[2] = {0, 0}, cr[2] = {0, 0};
      const float im = scale_inverse(sm), ir = scale_inverse(sr);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x = u4_word(draw, i >> 1) >> (16 * (i & 1)) & 0xFFFFu;
        const uint32_t y = (x >> 8) | ((x & 0xFFu) << 8);
        cm[i >> 2] |= round_m(m[i] * im, x) << (8 * (i & 3));
        cr[i >> 2] |= round_r(r[i] * ir, (v[i] * ir) * ir, y, v[i] > 0.f ? 1u : 0u) << (8 * (i & 3));
      }
      if (sm == 255u) cm[0] = cm[1] = 0;
      if (sr == 255u) cr[0] = cr[1] = 0;
      store_codes((uint8_t*)d.exp_avg_out, e, n, cm);
      store_codes((uint8_t*)d.exp_avg_sq_out, e, n, cr);
      if (n && (threadIdx.x & 3) == 0) {
        d.exp_avg_scale_out[e >> 5] = (uint8_t)sm;
        d.exp_avg_sq_scale_out[e >> 5] = (uint8_t)sr;
      }
    }
  }
}

// the 8-bit moments as the values they stand for (m, and v = r^2)
template <typename T>
__global__ __launch_bounds__(256) void adamw_values_kernel(const llp_adamw_desc* __restrict__ descs,
                                                           const int32_t* __restrict__ work, int64_t n_work) {
  for (int64_t w = blockIdx.x; w < n_work; w += gridDim.x) {
    const llp_adamw_desc d = descs[work[2 * w]];
    const int64_t e = (int64_t)work[2 * w + 1] * AW_ITEM + 8 * threadIdx.x;
    const int n = e >= d.numel ? 0 : (int)(d.numel - e < 8 ? d.numel - e : 8);
    if (!n) continue;
    uint32_t cm[2], cr[2];
    float m[8], r[8];
    load_codes((const uint8_t*)d.exp_avg_out, e, n, cm);
    load_codes((const uint8_t*)d.exp_avg_sq_out, e, n, cr);
    decode_m(cm, d.exp_avg_scale_out[e >> 5], m);
    decode_r(cr, d.exp_avg_sq_scale_out[e >> 5], r);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] *= r[i];
    if (d.exp_avg_value) store8<true>((T*)d.exp_avg_value, e, n, m);
    if (d.exp_avg_sq_value) store8<true>((T*)d.exp_avg_sq_value, e, n, r);
  }
}

// copy_t[c, r] = param_out[r, c], 64 x 64 tiles through LDS; work: (tensor, tile) pairs
template <typename P>
__global__ __launch_bounds__(256) void adamw_copy_t_kernel(const llp_adamw_desc* __restrict__ descs,
                                                           const int32_t* __restrict__ work) {
  __shared__ float tile[64][65];
  const llp_adamw_desc d = descs[work[2 * (int64_t)blockIdx.x]];
  if (!d.copy_t) return;
  const int64_t ti = work[2 * (int64_t)blockIdx.x + 1], tc = (d.cols + 63) / 64;
  const int64_t r0 = (ti / tc) * 64, c0 = (ti % tc) * 64;
  const int64_t ldt = d.copy_t_ld ? d.copy_t_ld : d.rows;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const P* p = (const P*)d.param_out;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = ty + 4 * j;
    const int64_t r = r0 + i, c = c0 + tx;
    if (r < d.rows && c < d.cols) {
      if constexpr (sizeof(P) == 4) tile[i][tx] = p[r * d.cols + c];
      else tile[i][tx] = bf2f(p[r * d.cols + c]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int i = ty + 4 * j;
    const int64_t c = c0 + i, r = r0 + tx;
    if (c < d.cols && r < d.rows) {
      if (d.copy_dtype == LLP_BF16) ((bf16_t*)d.copy_t)[c * ldt + r] = f2bf(tile[tx][i]);
      else ((float*)d.copy_t)[c * ldt + r] = tile[tx][i];
    }
  }
}

unsigned aw_grid(int64_t n_work) { return (unsigned)(n_work < 4096 ? n_work : 4096); }

bool known(int dtype) { return dtype == LLP_F32 || dtype == LLP_BF16; }

}  // namespace

extern "C" int64_t llp_adamw_work_items(int64_t numel) { return numel < 0 ? 0 : (numel + AW_ITEM - 1) / AW_ITEM; }

extern "C" int llp_adamw_step(const llp_adamw_desc* descs, int n_tensors, const int32_t* work, int64_t n_work,
                              int state_bits, int param_dtype, int grad_dtype, const float* sumsq, double max_norm,
                              double lr, double beta1, double beta2, double eps, double weight_decay,
                              const int64_t* step, uint64_t seed, void* stream) {
  LLP_CHECK_ARG(n_tensors >= 0 && n_tensors <= 65536 && n_work >= 0 && n_work < (1ll << 31),
                "llp_adamw_step: n_tensors in [0, 65536], n_work in [0, 2^31)");
  LLP_CHECK_ARG(state_bits == 32 || state_bits == 8, "llp_adamw_step: state_bits must be 32 or 8");
  LLP_CHECK_ARG(known(param_dtype) && known(grad_dtype), "llp_adamw_step: params and grads in f32 or bf16");
  LLP_CHECK_ARG(lr >= 0 && eps >= 0 && weight_decay >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1,
                "llp_adamw_step: lr, eps, weight_decay >= 0 and betas in [0, 1)");
  if (n_work == 0) return LLP_OK;
  LLP_CHECK_ARG(descs && work && step, "llp_adamw_step: null pointer");
  const AdamWArgs a{lr, beta1, beta2, eps, weight_decay, max_norm, seed};
  // Large steps: params, gradients and copies pass by the caches, which the moments then keep to themselves.  f32 moments
  // of more than 16 M elements, with a workgroup for every item: 2e7 elements 107 -> 96 us, 4e7 229 -> 222, 1e8 in place 589 -> 548
  // (1e7 would go from 46 to 50).  8-bit ones of more than 32 M, in 4,096 workgroups as always, for the step's constants and the
  // rounding take longer (1e8 340, one an item 347): 4e7 151 -> 140, 1e8 369 -> 340 (2e7 would go from 64 to 70).  With what reads
  // the params or the copies next the gain stays: the transposed copies' launch, f32 moments 2e7 136 -> 134, 4e7 296 -> 294, 1e8 826 ->
  // 769, 8-bit 4e7 215 -> 203, 1e8 620 -> 560; a read of the bf16 copy, f32 2e7 132 -> 110, 4e7 260 -> 260, 1e8 621 -> 625, 8-bit 4e7
  // 182 -> 171, 1e8 444 -> 446.
  const unsigned grid = state_bits == 32 && n_work > 8192 ? (unsigned)std::min<int64_t>(n_work, 1 << 20) : aw_grid(n_work);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, descs, work, n_work, sumsq, a, step);
  };
  auto types = [&](auto bits, auto once) {
    constexpr int B = bits;
    constexpr bool O = once;
    if (param_dtype == LLP_F32) grad_dtype == LLP_F32 ? go(adamw_kernel<B, O, float, float>) : go(adamw_kernel<B, O, float, bf16_t>);
    else grad_dtype == LLP_F32 ? go(adamw_kernel<B, O, bf16_t, float>) : go(adamw_kernel<B, O, bf16_t, bf16_t>);
  };
  constexpr std::integral_constant<int, 32> b32{};
  constexpr std::integral_constant<int, 8> b8{};
  if (state_bits == 32) n_work > 8192 ? types(b32, std::true_type{}) : types(b32, std::false_type{});
  else if (n_work >= 16384) types(b8, std::true_type{});
  else types(b8, std::false_type{});
  LLP_LAUNCH_CHECK();
  return LLP_OK;
}

extern "C" int llp_adamw_values(const llp_adamw_desc* descs, const int32_t* work, int64_t n_work, int dtype,
                                void* stream) {
  LLP_CHECK_ARG(known(dtype), "llp_adamw_values: values in f32 or bf16");
  LLP_CHECK_ARG(n_work >= 0 && n_work < (1ll << 31), "llp_adamw_values: n_work in [0, 2^31)");
  if (n_work == 0) return LLP_OK;
  LLP_CHECK_ARG(descs && work, "llp_adamw_values: null pointer");
  if (dtype == LLP_F32)
    hipLaunchKernelGGL(adamw_values_kernel<float>, dim3(aw_grid(n_work)), dim3(256), 0, (hipStream_t)stream, descs, work, n_work);
  else
    hipLaunchKernelGGL(adamw_values_kernel<bf16_t>, dim3(aw_grid(n_work)), dim3(256), 0, (hipStream_t)stream, descs, work, n_work);
  LLP_LAUNCH_CHECK();
  return LLP_OK;
}

extern "C" int64_t llp_adamw_copy_t_items(int64_t rows, int64_t cols) { return ((rows + 63) / 64) * ((cols + 63) / 64); }

extern "C" int llp_adamw_copy_t(const llp_adamw_desc* descs, const int32_t* work, int64_t n_work, int param_dtype,
                                void* stream) {
  LLP_CHECK_ARG(known(param_dtype), "llp_adamw_copy_t: params in f32 or bf16");
  LLP_CHECK_ARG(n_work >= 0 && n_work < (1ll << 31), "llp_adamw_copy_t: n_work in [0, 2^31)");
  if (n_work == 0) return LLP_OK;
  LLP_CHECK_ARG(descs && work, "llp_adamw_copy_t: null pointer");
  if (param_dtype == LLP_F32)
    hipLaunchKernelGGL(adamw_copy_t_kernel<float>, dim3((unsigned)n_work), dim3(256), 0, (hipStream_t)stream, descs, work);
  else
    hipLaunchKernelGGL(adamw_copy_t_kernel<bf16_t>, dim3((unsigned)n_work), dim3(256), 0, (hipStream_t)stream, descs, work);
  LLP_LAUNCH_CHECK();
  return LLP_OK;
}
