// What the differentiable layers share: the counter-based dropout mask, the activations with their derivatives, and
// loads / stores of eight consecutive columns of a row.
//
// The mask is a pure function of (seed, offset, row, column), so the forward pass, the backward pass and every fused
// epilogue recompute it and nothing is stored.  The generator is Philox4x32 with 10 rounds (Salmon, Moraes, Dror,
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11): key = seed, counter = (column / 8, row, row >> 32,
// offset).  One call gives four 32-bit words = eight 16-bit numbers, one per column 8 j .. 8 j + 7, low half first.
// Element kept if its number >= thr = round(p 65536); kept values are scaled by 65536 / (65536 - thr), the reciprocal
// of the probability that is really used, so the expectation is exact.  16 bits per element keep the generator
// below the memory time: a call is about 480 cycles of a wave (20 quarter-rate multiplies, 20 three-input XORs), half of
// what eight 16-bit elements per lane take to come from and go to HBM; 32 bits per element would take as long as they do.
#pragma once
#include "common.h"

struct DropArgs {
  unsigned thr;                 // 0: no dropout, 65536: everything dropped
  float scale;
  unsigned k0, k1;              // seed
  const unsigned* seed_dev;     // not null: the seed's two words are read there instead (low word first)
  unsigned offset;
};

// p and the counter's host-side words -> DropArgs; refuses what is no probability and offsets beyond 32 bits
static inline int drop_args(DropArgs* d, double p, int64_t seed, const int64_t* seed_dev, int64_t offset, const char* who) {
  SDMI_REQUIRE(p >= 0.0 && p <= 1.0, "%s: p = %g is no probability", who, p);
  SDMI_REQUIRE(offset >= 0 && offset <= 0xFFFFFFFFll, "%s: offset %lld does not fit 32 bits", who, (long long)offset);
  SDMI_REQUIRE(((uintptr_t)seed_dev & 7) == 0, "%s: the seed in device memory must be 8-byte aligned", who);
  const double t = __builtin_nearbyint(p * 65536.0);
  d->thr = (unsigned)t;
  d->scale = d->thr < 65536u ? (float)(65536.0 / (65536.0 - t)) : 0.f;
  d->k0 = (unsigned)((uint64_t)seed & 0xFFFFFFFFu); d->k1 = (unsigned)((uint64_t)seed >> 32);
  d->seed_dev = (const unsigned*)seed_dev;
  d->offset = (unsigned)offset;
  return SDMI_OK;
}

enum { ACT_NONE = 0, ACT_SILU = 1, ACT_GELU = 2, ACT_QUICK_GELU = 3, ACT_COUNT = 4 };

#ifdef __HIPCC__
__device__ __forceinline__ void drop_key(const DropArgs& d, unsigned& k0, unsigned& k1) {
  k0 = d.k0; k1 = d.k1;
  if (d.seed_dev) { k0 = d.seed_dev[0]; k1 = d.seed_dev[1]; }
}

__device__ __forceinline__ unsigned xor3(unsigned a, unsigned b, unsigned c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}
struct Keep8 { unsigned w[4]; };     // 16-bit number of column e: half (e & 1) of word e / 2

__device__ __forceinline__ Keep8 philox8(unsigned k0, unsigned k1, unsigned col8, uint64_t row, unsigned offset) {
  unsigned c0 = col8, c1 = (unsigned)row, c2 = (unsigned)(row >> 32), c3 = offset;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = xor3((unsigned)(b >> 32), c1, k0);
    c2 = xor3((unsigned)(a >> 32), c3, k1);
    c1 = (unsigned)b;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  return Keep8{{c0, c1, c2, c3}};
}
// whether column e (of 8) is kept: the high half compares in place, the low one shifted up; thr16 = thr << 16 (thr < 65536)
__device__ __forceinline__ bool keeps(const Keep8& k, int e, unsigned thr16) {
  return ((e & 1) ? k.w[e >> 1] : k.w[e >> 1] << 16) >= thr16;
}
// dropped elements are zero whatever they held (infinities and NaN included); thr = 65536 keeps none
__device__ __forceinline__ void drop8(float (&v)[8], const Keep8& k, unsigned thr, float scale) {
  if (thr > 65535u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = keeps(k, e, thr << 16) ? v[e] * scale : 0.f;
}

// ---- activations ---------------------------------------------------------------------------------
// fp32 tensors take the library functions, or (sigmoid) as good as those; 16-bit ones the hardware exponential (relative
// error a few 2^-23, times the exponent's size) and, for the normal distribution function of GELU, e^{-x^2} t P(t) with
// t = 1 / (1 + 0.43 x) and P of degree 7: a fit of erfc(x) e^{x^2} / 2 on 0 <= x <= 10 by Lawson's reweighted least squares,
// whose error is relative (1e-7, 4e-7 as evaluated), so that the tail that GELU shows below -3 keeps all the digits of 16
// bits; one exponential gives the density for the derivative too.
// e^-x reaches infinity below x = -88, where the reciprocal is 0
template <typename T> __device__ __forceinline__ float sigmoid_for(float x) {
  if constexpr (sizeof(T) == 4) {
    // e^-x as 2^t (1 + r ln 2) with t + r = -x log2 e, r what the product's rounding and the constant's lose: an ulp or two
    // for a handful of instructions.  x stops at +-88 (t and 2^t finite); a NaN passes through the selects
    const float lo = x < -88.f ? -88.f : x, y = lo > 88.f ? 88.f : lo;
    const float t = -y * 1.44269502162933349609375f;
    const float r = fmaf(-y, 1.925963033500011e-08f, fmaf(-y, 1.44269502162933349609375f, -t));
    const float p = __builtin_amdgcn_exp2f(t);
    return __builtin_amdgcn_rcpf(1.f + fmaf(p, r * 0.693147182464599609375f, p));
  } else {
    return __builtin_amdgcn_rcpf(1.f + __expf(-x));
  }
}
// Phi(z) and, on demand, the density phi(z)
template <typename T> __device__ __forceinline__ float normal_cdf(float z, float* pdf) {
  if constexpr (sizeof(T) == 4) {
    if (pdf) *pdf = 0.39894228040143267794f * expf(-0.5f * z * z);
    return 0.5f * erfcf(-z * 0.70710678118654752440f);
  } else {
    const float x = fabsf(z) * 0.70710678118654752440f;
    const float ex = __expf(-x * x);
    if (pdf) *pdf = 0.39894228040143267794f * ex;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.43f, x, 1.f));
    float q = fmaf(0.0365728475f, t, -0.154047564f);
    q = fmaf(q, t, 0.189943194f);
    q = fmaf(q, t, -0.0411517546f);
    q = fmaf(q, t, 0.122540131f);
    q = fmaf(q, t, 0.102736309f);
    q = fmaf(q, t, 0.122146904f);
    q = fmaf(q, t, 0.121259913f);
    q = q * t * ex;                              // upper tail beyond |z|
    return z < 0.f ? q : 1.f - q;
  }
}
// z g with z -> -inf, g -> 0 would be NaN where the limit is 0: the factor z stops at -1e4, where g has long been 0 (the
// gate still sees z itself, so a NaN stays one)
template <typename T, int N> __device__ __forceinline__ void act_n(float (&z)[N], int act) {
  if (act == ACT_NONE) return;
  if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) z[e] = fmaxf(z[e], -1e4f) * normal_cdf<T>(z[e], nullptr);
  } else {
    const float a = act == ACT_QUICK_GELU ? 1.702f : 1.f;
#pragma unroll
    for (int e = 0; e < N; ++e) z[e] = fmaxf(z[e], -1e4f) * sigmoid_for<T>(a * z[e]);
  }
}
// g[e] *= act'(z[e])
template <typename T, int N> __device__ __forceinline__ void act_grad_n(const float (&z)[N], float (&g)[N], int act) {
  if (act == ACT_NONE) return;
  if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float pdf;
      const float cdf = normal_cdf<T>(z[e], &pdf);
      g[e] *= fmaf(__builtin_amdgcn_fmed3f(z[e], -1e4f, 1e4f), pdf, cdf);
    }
  } else {
    const float a = act == ACT_QUICK_GELU ? 1.702f : 1.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float s = sigmoid_for<T>(a * z[e]);
      g[e] *= fmaf(a * __builtin_amdgcn_fmed3f(z[e], -1e4f, 1e4f) * s, 1.f - s, s);
    }
  }
}

// ---- eight columns of a row ------------------------------------------------------------------------
// Whole groups go as 16-byte accesses that assume element alignment only (the hardware takes any dword or half
// address); a row's last group, if it is short, goes element by element.
template <typename T> struct Vec8u {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <typename T> __device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    const typename Vec8u<T>::type r = *reinterpret_cast<const typename Vec8u<T>::type*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(r[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? to_f32<T>(p[e]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    typename Vec8u<T>::type r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = from_f32<T>(v[e]);
    *reinterpret_cast<typename Vec8u<T>::type*>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = from_f32<T>(v[e]);
  }
}

#endif

// n / d for 0 <= n < 2^31 by one multiply-high (d >= 1): division by an invariant, Granlund and Montgomery 1994
struct FastDiv { unsigned mul, shift, d; };
static inline FastDiv fast_div(unsigned d) {
  FastDiv f{0, 0, d};
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = (unsigned)((((1ull << f.shift) - d) << 32) / d + 1);
  return f;
}
#ifdef __HIPCC__
__device__ __forceinline__ unsigned div_by(unsigned n, const FastDiv& f) { return (__umulhi(n, f.mul) + n) >> f.shift; }
#endif
