// GroupNorm with activation and dropout, channels last, and its gradients:
//   xh = (x - mean_g) rstd_g      u = gamma xh + beta        y = drop(act(u))
//   du = drop(dy) act'(u)         dgamma = sum du xh         dbeta = sum du        h = gamma du
//   dx = rstd_g (h - mean_g(h) - xh mean_g(h xh))            (means over the sample's group)
// The input may be the channel concatenation of two tensors; any channel count per group, any image size.
//
// A (sample, group) slice that fits LDS is one workgroup's work: read once, normalised from LDS, one launch (the
// weight gradients of several samples take a second one).  Larger slices take two launches over strips of pixels:
// the first leaves per-strip sums, the second folds them in double and finishes the strip.  Every sum is taken in a
// fixed order.  Statistics never go through E[x^2] - E[x]^2, where a common offset or an outlier a (feature maps have them, in
// corners too) leaves the rounding of a^2 in a variance that may be a^2 / n.  A slice takes two passes over LDS.  A thread
// of a strip updates its columns' running means and squares about them (Welford 1962); a group's threads and columns, and
// then the strips, are joined by the squares of their means' distances from the joint mean (Chan, Golub, LeVeque 1979).
//
// Bounds, MI355X, 16x64x64x320 bf16 (42 MB a tensor) with SiLU and dropout: statistics 13 us (HBM: 8), apply 22, gradient
// sums 22, gradient apply 24 us.  The last three are the vector ALU's: a wave spends about 1100 cycles on the generator
// (480) and the SiLU (its exponential and reciprocal at a quarter of the rate) of 512 elements, 20 us in all, where HBM
// would take 16, 16 and 24.  3x37x53x480 fp32: 8, 10, 9 and 10 us, launches and the fold of the strips.  One workgroup per
// slice: 2x8x8x1280 fp16 forward 5.8 us, a launch; 16x16x16x1280 bf16 12 forward, 19 + 4 backward (HBM: 4 and 6): 512 workgroups,
// one round of two per CU, whose load, three sums over the workgroup and store wait for one another.
#include "act_drop.h"
#include "ops.h"
#include <stdio.h>

namespace {

constexpr unsigned SLICES_X = 1u << 20;      // slices of a row of the grid: a launch has less than 2^32 threads that way
constexpr int GNA_MAX_C = 8192;               // a thread per eight channels, and their sums fit LDS

struct GnaParams {
  const void* x0; const void* x1; const void* dy;
  void* out0; void* out1;                     // forward: out0 = y [B][HW][C]; backward: dx of x0, x1
  int c0, c1, C, G, cpg, B;
  int64_t HW;
  FastDiv div_cpg;
  float eps;
  const float* gamma; const float* beta;
  int act;
  DropArgs drop;
  float* stats;                               // [B][G][2]: mean, rstd
  int strips; int64_t px_per_strip;
  float* part;                                // [B][strips][G][2] of a strip's groups: mean and squares about it; backward sums
  float* cpart;                               // backward: [B][strips][2][C] sums of a strip's channels
  float* dgamma; float* dbeta;
  int apply_blocks;                           // backward: blockIdx.x beyond fold dgamma / dbeta
};

// columns c .. c + W - 1 (of C) of pixel row `row` of the two-source tensor
template <typename T, int W>
__device__ __forceinline__ void load_n(const T* p, float (&v)[W]) {
  if constexpr (W == 8) load8<T>(p, 8, v);
  else {
    typedef T V __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    if constexpr (W == 1) v[0] = to_f32<T>(*p);
    else {
      const V r = *reinterpret_cast<const V*>(p);
#pragma unroll
      for (int e = 0; e < W; ++e) v[e] = to_f32<T>(r[e]);
    }
  }
}
template <typename T, int W>
__device__ __forceinline__ void store_n(T* p, const float (&v)[W]) {
  if constexpr (W == 8) store8<T>(p, 8, v);
  else if constexpr (W == 1) *p = from_f32<T>(v[0]);
  else {
    typedef T V __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    V r;
#pragma unroll
    for (int e = 0; e < W; ++e) r[e] = from_f32<T>(v[e]);
    *reinterpret_cast<V*>(p) = r;
  }
}
// Eight columns of a two-source tensor that a thread walks down, from row `row0` on.  WHOLE: all groups of eight lie in one
// source, 16-byte pieces (32 in fp32) that stay packed until they are used; otherwise every group goes element by element, as a
// row's short last group and one that straddles the sources must.
template <typename T, bool WHOLE> struct Cols;
template <typename T> struct Cols<T, true> {
  typedef T Raw __attribute__((ext_vector_type(8)));
  char* p;
  unsigned step;                  // bytes from row to row
  __device__ __forceinline__ Cols(const void* x0, const void* x1, int c0, int c1, int c, int64_t row0) {
    const bool second = c >= c0;
    step = (unsigned)(second ? c1 : c0) * (unsigned)sizeof(T);
    p = (char*)(second ? x1 : x0) + row0 * step + (second ? c - c0 : c) * (int)sizeof(T);
  }
  __device__ __forceinline__ Raw load(int r) const {
    return *reinterpret_cast<const typename Vec8u<T>::type*>(p + (unsigned)r * step);
  }
  __device__ __forceinline__ void store(int r, const float (&v)[8]) const {
    store8<T>(reinterpret_cast<T*>(p + (unsigned)r * step), 8, v);
  }
};
template <typename T> struct Cols<T, false> {
  typedef T Raw __attribute__((ext_vector_type(8)));
  T* p0; T* p1;                   // element 0 of row row0 in each source (the columns' own offset included)
  int c0, c1, n0, n;              // row strides; elements in the first source, in both
  __device__ __forceinline__ Cols(const void* x0, const void* x1, int c0_, int c1_, int c, int64_t row0) : c0(c0_), c1(c1_) {
    const int left = c0 - c, all = c0 + c1 - c;
    n0 = left < 0 ? 0 : (left < 8 ? left : 8);
    n = all < 8 ? all : 8;
    p0 = (T*)x0 + row0 * c0 + c;
    p1 = (T*)x1 + row0 * c1 - left;
  }
  __device__ __forceinline__ Raw load(int64_t r) const {
    Raw v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n0 ? p0[r * c0 + e] : (e < n ? p1[r * c1 + e] : (T)0.f);
    return v;
  }
  __device__ __forceinline__ void store(int64_t r, const float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < n0) p0[r * c0 + e] = from_f32<T>(v[e]);
      else if (e < n) p1[r * c1 + e] = from_f32<T>(v[e]);
    }
  }
};
// per-channel fp32 parameters of eight columns (the last one repeated beyond the row)
__device__ __forceinline__ void load_params(const float* p, int c, int C, float (&v)[8]) {
  if (c + 8 <= C) load8<float>(p + c, 8, v);
  else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = p[c + e < C ? c + e : C - 1];
  }
}
// W columns from c on, that do not leave their group of eight
template <int W>
__device__ __forceinline__ void drop_n(const DropArgs& d, unsigned k0, unsigned k1, int64_t row, int c, float (&v)[W]) {
  if (!d.thr) return;
  const Keep8 k = philox8(k0, k1, (unsigned)c >> 3, (uint64_t)row, d.offset);
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const int ce = (c & (8 - W)) + e;
    const unsigned wd = ce < 4 ? (ce < 2 ? k.w[0] : k.w[1]) : (ce < 6 ? k.w[2] : k.w[3]);
    v[e] = ((ce & 1) ? wd >> 16 : wd & 0xFFFFu) >= d.thr ? v[e] * d.scale : 0.f;
  }
}

// ---- one workgroup per (sample, group) ---------------------------------------------------------------
__device__ __forceinline__ float block_sum(float v, float* red) {       // red: 16 floats; same value on every thread
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
  for (unsigned w = 0; w < blockDim.x >> 6; ++w) t += red[w];
  return t;
}
__device__ __forceinline__ bool slice_of_block(const GnaParams& p, int& b, int& g) {
  // neighbouring groups of a sample share 128-byte lines: a contiguous run of slices per XCD
  const unsigned block = blockIdx.y * SLICES_X + blockIdx.x;
  const unsigned total = (unsigned)p.B * (unsigned)p.G, xcd = block & 7, q8 = total >> 3, r8 = total & 7;
  const unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (block >> 3);
  b = (int)(id / (unsigned)p.G); g = (int)(id - (unsigned)b * (unsigned)p.G);
  return block < total;
}

template <typename T, int W>
__global__ __launch_bounds__(1024) void gna_slice_fwd_kernel(GnaParams p) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[16];
  T* xs = reinterpret_cast<T*>(smem);
  int b, g;
  if (!slice_of_block(p, b, g)) return;
  const int cbase = g * p.cpg, vpp = p.cpg / W, nv = (int)p.HW * vpp;
  float s = 0.f;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    const int px = (int)div_by((unsigned)i, p.div_cpg), c = cbase + (i - px * vpp) * W;
    const int64_t row = (int64_t)b * p.HW + px;
    float v[W];
    if (c < p.c0) load_n<T, W>((const T*)p.x0 + row * p.c0 + c, v);
    else load_n<T, W>((const T*)p.x1 + row * p.c1 + (c - p.c0), v);
    store_n<T, W>(xs + i * W, v);
#pragma unroll
    for (int e = 0; e < W; ++e) s += v[e];
  }
  const float inv_n = 1.f / ((float)p.HW * (float)p.cpg);
  const float m0 = block_sum(s, red) * inv_n;
  float q = 0.f, d = 0.f;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {      // a thread reads back what it wrote
    float v[W];
    load_n<T, W>(xs + i * W, v);
#pragma unroll
    for (int e = 0; e < W; ++e) { const float t = v[e] - m0; d += t; q = fmaf(t, t, q); }
  }
  d = block_sum(d, red) * inv_n;                            // what the first sum's rounding left over
  const float var = fmaxf(block_sum(q, red) * inv_n - d * d, 0.f);
  const float mean = m0 + d, rstd = 1.f / sqrtf(var + p.eps);
  if (threadIdx.x == 0) {
    p.stats[((size_t)b * p.G + g) * 2] = mean;
    p.stats[((size_t)b * p.G + g) * 2 + 1] = rstd;
  }
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    const int px = (int)div_by((unsigned)i, p.div_cpg), c = cbase + (i - px * vpp) * W;
    const int64_t row = (int64_t)b * p.HW + px;
    float v[W];
    load_n<T, W>(xs + i * W, v);
#pragma unroll
    for (int e = 0; e < W; ++e) v[e] = fmaf(v[e] - mean, rstd * p.gamma[c + e], p.beta[c + e]);
    act_n<T>(v, p.act);
    drop_n<W>(p.drop, k0, k1, row, c, v);
    store_n<T, W>((T*)p.out0 + row * p.C + c, v);
  }
}

// du of W columns from x and dy
template <typename T, int W>
__device__ __forceinline__ void grad_u(const GnaParams& p, unsigned k0, unsigned k1, int64_t row, int c, float mean, float rstd,
                                       const float (&x)[W], const float (&dy)[W], float (&xh)[W], float (&du)[W]) {
  float u[W];
#pragma unroll
  for (int e = 0; e < W; ++e) {
    xh[e] = (x[e] - mean) * rstd;
    u[e] = fmaf(xh[e], p.gamma[c + e], p.beta[c + e]);
    du[e] = dy[e];
  }
  drop_n<W>(p.drop, k0, k1, row, c, du);
  act_grad_n<T>(u, du, p.act);
}

// Backward of a slice: x and du stay in LDS from the group's sums to dx and the channels' sums.
template <typename T, int W>
__global__ __launch_bounds__(1024) void gna_slice_bwd_kernel(GnaParams p) {
  extern __shared__ __align__(16) char smem[];
  __shared__ float red[16];
  int b, g;
  if (!slice_of_block(p, b, g)) return;
  const int cbase = g * p.cpg, vpp = p.cpg / W, nv = (int)p.HW * vpp;
  float* dus = reinterpret_cast<float*>(smem);                     // [HW][cpg] fp32
  T* xs = reinterpret_cast<T*>(smem + (size_t)p.HW * p.cpg * 4);   // [HW][cpg]
  const float mean = p.stats[((size_t)b * p.G + g) * 2], rstd = p.stats[((size_t)b * p.G + g) * 2 + 1];
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  float a1 = 0.f, a2 = 0.f;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    const int px = (int)div_by((unsigned)i, p.div_cpg), c = cbase + (i - px * vpp) * W;
    const int64_t row = (int64_t)b * p.HW + px;
    float x[W], dy[W], xh[W], du[W];
    if (c < p.c0) load_n<T, W>((const T*)p.x0 + row * p.c0 + c, x);
    else load_n<T, W>((const T*)p.x1 + row * p.c1 + (c - p.c0), x);
    load_n<T, W>((const T*)p.dy + row * p.C + c, dy);
    grad_u<T, W>(p, k0, k1, row, c, mean, rstd, x, dy, xh, du);
    store_n<T, W>(xs + i * W, x);
    store_n<float, W>(dus + i * W, du);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float h = du[e] * p.gamma[c + e];
      a1 += h;
      a2 = fmaf(h, xh[e], a2);
    }
  }
  const float inv_n = 1.f / ((float)p.HW * (float)p.cpg);
  a1 = block_sum(a1, red) * inv_n;
  a2 = block_sum(a2, red) * inv_n;                                 // (its barriers also make xs and dus visible)
  if (p.out0 || p.out1) {
    for (int i = threadIdx.x; i < nv; i += blockDim.x) {
      const int px = (int)div_by((unsigned)i, p.div_cpg), c = cbase + (i - px * vpp) * W;
      const int64_t row = (int64_t)b * p.HW + px;
      float x[W], du[W];
      load_n<T, W>(xs + i * W, x);
      load_n<float, W>(dus + i * W, du);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float xh = (x[e] - mean) * rstd;
        x[e] = rstd * (du[e] * p.gamma[c + e] - a1 - xh * a2);
      }
      if (c < p.c0) { if (p.out0) store_n<T, W>((T*)p.out0 + row * p.c0 + c, x); }
      else if (p.out1) store_n<T, W>((T*)p.out1 + row * p.c1 + (c - p.c0), x);
    }
  }
  if (!p.dgamma && !p.dbeta) return;
  // channel sums over the pixels: a wave per channel, its lanes' sums folded by shuffles
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  for (int c = wave; c < p.cpg; c += nw) {
    float s1 = 0.f, s2 = 0.f;
    for (int px = lane; px < (int)p.HW; px += 64) {
      const float du = dus[px * p.cpg + c];
      s1 += du;
      s2 = fmaf(du, (to_f32<T>(xs[px * p.cpg + c]) - mean) * rstd, s2);
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (lane == 0) {
      if (p.B == 1) {
        if (p.dbeta) p.dbeta[cbase + c] = s1;
        if (p.dgamma) p.dgamma[cbase + c] = s2;
      } else {
        p.cpart[((size_t)b * 2) * p.C + cbase + c] = s1;
        p.cpart[((size_t)b * 2 + 1) * p.C + cbase + c] = s2;
      }
    }
  }
}

// ---- strips ------------------------------------------------------------------------------------------
// A thread owns one group of eight columns (a block has at least as many threads) and walks every lanes-th pixel of its
// strip.
// pixels a thread has in flight while it works on as many: 64 bytes (32 of each tensor backward), what the registers hold
template <typename T> struct Depth { static constexpr int FWD = 16 / (int)sizeof(T) / 2, BWD = 1; };
struct Walk { int ncg, lanes, pl, cg, count; int64_t row0; bool live; };      // count pixels from row row0 on
__device__ __forceinline__ Walk walk_of(const GnaParams& p, int strip, int b) {
  Walk w;
  w.ncg = (p.C + 7) >> 3;
  w.lanes = (int)blockDim.x / w.ncg;
  w.pl = (int)threadIdx.x / w.ncg;
  w.cg = (int)threadIdx.x - w.pl * w.ncg;
  w.live = w.pl < w.lanes;                               // the others are left over
  const int64_t pb = (int64_t)strip * p.px_per_strip, left = p.HW - pb;
  w.count = (int)(left < p.px_per_strip ? left : p.px_per_strip);
  w.row0 = (int64_t)b * p.HW + pb;
  return w;
}
// the pixels px, px + lanes, ... of a walk (beyond the strip its last one again, which the caller does not count)
template <typename C, int N>
__device__ __forceinline__ void fetch(const C& x, const Walk& w, int px, typename C::Raw (&r)[N]) {
#pragma unroll
  for (int u = 0; u < N; ++u) r[u] = x.load(min(px + u * w.lanes, w.count - 1));
}
// threads per group for folds over the groups: a power of two, at most a wave
__device__ __forceinline__ int threads_per_group(int G) {
  int t = 64;
  while (t > 1 && t * G > (int)blockDim.x) t >>= 1;
  return t;
}
template <typename F> __device__ __forceinline__ F fold_lanes(F v, int tpg) {
  for (int o = tpg >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// the strip's channel sums in LDS ([lanes][ncg * 8], two arrays) -> lane 0's row holds the totals
__device__ __forceinline__ void fold_pixel_lanes(float* s1, float* s2, int lanes, int width) {
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += (int)blockDim.x) {
    float a = s1[c], q = s2[c];
    for (int l = 1; l < lanes; ++l) { a += s1[l * width + c]; q += s2[l * width + c]; }
    s1[c] = a; s2[c] = q;
  }
  __syncthreads();
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(1024) void gna_stats_kernel(GnaParams p) {
  constexpr int WALK = Depth<T>::FWD;
  extern __shared__ __align__(16) char smem[];
  const int strip = blockIdx.x, b = blockIdx.y;
  const Walk w = walk_of(p, strip, b);
  typedef Cols<T, WHOLE> C;
  const int width = w.ncg * 8;
  float* s_mean = reinterpret_cast<float*>(smem);      // [lanes][width] each
  float* s_sq = s_mean + w.lanes * width;
  const int c = w.cg * 8;
  const C x(p.x0, p.x1, p.c0, p.c1, c, w.row0);
  typename C::Raw r[WALK];
  if (w.live) {
    fetch(x, w, w.pl, r);
    float mean[8], sq[8], n = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { mean[e] = 0.f; sq[e] = 0.f; }
    for (int px = w.pl; px < w.count; px += WALK * w.lanes) {
#pragma unroll
      for (int u = 0; u < WALK; ++u) {
        if (px + u * w.lanes >= w.count) break;
        n += 1.f;
        const float inv = __builtin_amdgcn_rcpf(n);    // within an ulp, a rounding like the others (and 1 / 1 is 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = to_f32<T>(r[u][e]), d = v - mean[e];
          mean[e] = fmaf(d, inv, mean[e]);
          sq[e] = fmaf(d, v - mean[e], sq[e]);
        }
      }
      if (px + WALK * w.lanes < w.count) fetch(x, w, px + WALK * w.lanes, r);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) { s_mean[w.pl * width + c + e] = mean[e]; s_sq[w.pl * width + c + e] = sq[e]; }
  }
  __syncthreads();
  // a group's lanes and columns: the joint mean about the first of them, then all squares about that
  const int tpg = threads_per_group(p.G), j = threadIdx.x & (tpg - 1);
  const int lanes = min(w.lanes, w.count), every = w.count / w.lanes, more = w.count - every * w.lanes;    // pixels: every, or one more
  const int l0 = j / p.cpg, dl = tpg / p.cpg, k0 = j - l0 * p.cpg, dk = tpg - dl * p.cpg;
  const float inv_n = 1.f / ((float)w.count * (float)p.cpg);
  for (int g0 = 0; g0 < p.G; g0 += (int)blockDim.x / tpg) {                // every lane goes round equally often (shuffles)
    const int g = g0 + (int)threadIdx.x / tpg;
    auto each = [&](auto fn) {       // fn(pixels, mean, squares about it) of this thread's share of lanes x columns
      for (int l = l0, k = k0; l < lanes;) {
        const int i = l * width + g * p.cpg + k;
        fn((float)(every + (l < more ? 1 : 0)), s_mean[i], s_sq[i]);
        l += dl; k += dk;
        if (k >= p.cpg) { k -= p.cpg; ++l; }
      }
    };
    float at = 0.f, a = 0.f;
    if (g < p.G) {
      at = s_mean[g * p.cpg];
      each([&](float n, float m, float) { a = fmaf(n, m - at, a); });
    }
    at = fmaf(fold_lanes(a, tpg), inv_n, at);
    float d = 0.f, q = 0.f;
    if (g < p.G)
      each([&](float n, float m, float sq) {
        const float t = m - at;
        d = fmaf(n, t, d);                             // what the first sum's rounding left over
        q += fmaf(n * t, t, sq);
      });
    d = fold_lanes(d, tpg) * inv_n;
    q = fold_lanes(q, tpg);
    if (g < p.G && j == 0) {
      float* dst = p.part + (((size_t)b * p.strips + strip) * p.G + g) * 2;
      dst[0] = at + d;
      q -= d * d * (float)w.count * (float)p.cpg;
      dst[1] = q < 0.f ? 0.f : q;                      // (a NaN stays)
    }
  }
}

// sums over the strips of sample b, per group, in double, of add's two terms of a strip's pair (and of the first strip's first
// number): fin(g, that number, first sum, second sum) on one thread per group
template <typename Add, typename Fn> __device__ __forceinline__ void fold_strips(const GnaParams& p, int b, Add add, Fn fin) {
  const int tpg = threads_per_group(p.G), j = threadIdx.x & (tpg - 1);
  for (int g0 = 0; g0 < p.G; g0 += (int)blockDim.x / tpg) {
    const int g = g0 + (int)threadIdx.x / tpg;
    double a = 0.0, q = 0.0, at = 0.0;
    if (g < p.G) {
      const float2* src = reinterpret_cast<const float2*>(p.part) + (size_t)b * p.strips * p.G + g;
      at = (double)src[0].x;
      for (int s0 = j; s0 < p.strips; s0 += 8 * tpg) {       // eight loads in flight, the ones beyond the end count nothing
        float2 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = src[(size_t)min(s0 + u * tpg, p.strips - 1) * p.G];
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (s0 + u * tpg < p.strips) add(s0 + u * tpg, at, v[u], a, q);
      }
    }
    a = fold_lanes(a, tpg);
    q = fold_lanes(q, tpg);
    if (g < p.G && j == 0) fin(g, at, a, q);
  }
}

template <typename T, int ACT, bool DROP, bool WHOLE>
__global__ __launch_bounds__(1024) void gna_apply_kernel(GnaParams p) {
  constexpr int WALK = Depth<T>::FWD;
  const int act = ACT < 0 ? p.act : ACT;
  extern __shared__ __align__(16) char smem[];
  float* s_mean = reinterpret_cast<float*>(smem);
  float* s_rstd = s_mean + p.G;
  const int strip = blockIdx.x, b = blockIdx.y;
  const Walk w = walk_of(p, strip, b);
  typedef Cols<T, WHOLE> C;
  typename C::Raw r[WALK];                     // the first pixels come while the strips' sums are folded
  const int c = w.cg * 8;
  const C x(p.x0, p.x1, p.c0, p.c1, c, w.row0);
  if (w.live) fetch(x, w, w.pl, r);
  const double n_strip = (double)p.px_per_strip * (double)p.cpg, n = (double)p.HW * (double)p.cpg;
  fold_strips(p, b, [&](int s, double at, float2 v, double& a, double& q) {
    const double w = s < p.strips - 1 ? n_strip : n - n_strip * (double)(p.strips - 1), d = (double)v.x - at;
    a += w * d;
    q += (double)v.y + w * d * d;
  }, [&](int g, double at, double a, double q) {
    const double m = a / n;
    double var = q / n - m * m;
    if (var < 0.0) var = 0.0;
    const float mean = (float)(at + m), rstd = (float)(1.0 / sqrt(var + (double)p.eps));
    s_mean[g] = mean; s_rstd[g] = rstd;
    if (strip == 0) {
      p.stats[((size_t)b * p.G + g) * 2] = mean;
      p.stats[((size_t)b * p.G + g) * 2 + 1] = rstd;
    }
  });
  __syncthreads();
  unsigned k0 = 0, k1 = 0;
  if (DROP) drop_key(p.drop, k0, k1);
  if (w.live) {
    const C y(p.out0, p.out0, p.C, 0, c, w.row0);
    float mn[8], sc[8], bt[8];
    load_params(p.gamma, c, p.C, sc);
    load_params(p.beta, c, p.C, bt);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int g = (int)div_by((unsigned)(c + e < p.C ? c + e : p.C - 1), p.div_cpg);
      mn[e] = s_mean[g]; sc[e] *= s_rstd[g];
    }
    for (int px = w.pl; px < w.count; px += WALK * w.lanes) {
      typename C::Raw now[WALK];
#pragma unroll
      for (int u = 0; u < WALK; ++u) now[u] = r[u];
      if (px + WALK * w.lanes < w.count) fetch(x, w, px + WALK * w.lanes, r);
#pragma unroll
      for (int u = 0; u < WALK; ++u) {
        if (px + u * w.lanes >= w.count) break;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(to_f32<T>(now[u][e]) - mn[e], sc[e], bt[e]);
        act_n<T>(v, act);
        if (DROP) drop8(v, philox8(k0, k1, (unsigned)w.cg, (uint64_t)(w.row0 + px + u * w.lanes), p.drop.offset), p.drop.thr, p.drop.scale);
        y.store(px + u * w.lanes, v);
      }
    }
  }
}

// backward, first launch: channel sums of du and du xh over the strip, and the group sums of gamma times them
template <typename T, int ACT, bool DROP, bool WHOLE>
__global__ __launch_bounds__(1024) void gna_grad_sums_kernel(GnaParams p) {
  constexpr int WALK_BWD = Depth<T>::BWD;
  const int act = ACT < 0 ? p.act : ACT;
  extern __shared__ __align__(16) char smem[];
  const int strip = blockIdx.x, b = blockIdx.y;
  const Walk w = walk_of(p, strip, b);
  typedef Cols<T, WHOLE> C;
  const int width = w.ncg * 8;
  float* s1 = reinterpret_cast<float*>(smem);
  float* s2 = s1 + w.lanes * width;
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  if (w.live) {
    const int c = w.cg * 8;
    const C x(p.x0, p.x1, p.c0, p.c1, c, w.row0), dy(p.dy, p.dy, p.C, 0, c, w.row0);
    typename C::Raw rx[WALK_BWD], rd[WALK_BWD];
    fetch(x, w, w.pl, rx);
    fetch(dy, w, w.pl, rd);
    // u = (x - mean) sc + beta with sc = rstd gamma; the sums take (x - mean) and the unscaled mask, rstd and the
    // dropout's scale come in at the end
    float mn[8], rs[8], sc[8], bt[8], s[8], q[8];
    load_params(p.gamma, c, p.C, sc);
    load_params(p.beta, c, p.C, bt);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* st = p.stats + ((size_t)b * p.G + (int)div_by((unsigned)(c + e < p.C ? c + e : p.C - 1), p.div_cpg)) * 2;
      mn[e] = st[0]; rs[e] = st[1];
      sc[e] *= rs[e];
      s[e] = 0.f; q[e] = 0.f;
    }
    for (int px = w.pl; px < w.count; px += WALK_BWD * w.lanes) {
      typename C::Raw nx[WALK_BWD], nd[WALK_BWD];
#pragma unroll
      for (int u = 0; u < WALK_BWD; ++u) { nx[u] = rx[u]; nd[u] = rd[u]; }
      if (px + WALK_BWD * w.lanes < w.count) {
        fetch(x, w, px + WALK_BWD * w.lanes, rx);
        fetch(dy, w, px + WALK_BWD * w.lanes, rd);
      }
#pragma unroll
      for (int u = 0; u < WALK_BWD; ++u) {
        if (px + u * w.lanes >= w.count) break;
        const int64_t row = w.row0 + px + u * w.lanes;
        float v[8], d[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = to_f32<T>(nd[u][e]);
          d[e] = to_f32<T>(nx[u][e]) - mn[e];
          z[e] = fmaf(d[e], sc[e], bt[e]);
        }
        if (DROP) drop8(v, philox8(k0, k1, (unsigned)w.cg, (uint64_t)row, p.drop.offset), p.drop.thr, 1.f);
        act_grad_n<T>(z, v, act);
#pragma unroll
        for (int e = 0; e < 8; ++e) { s[e] += v[e]; q[e] = fmaf(v[e], d[e], q[e]); }
      }
    }
    const float ds = DROP ? p.drop.scale : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) { s[e] *= ds; q[e] *= ds * rs[e]; }
#pragma unroll
    for (int e = 0; e < 8; ++e) { s1[w.pl * width + c + e] = s[e]; s2[w.pl * width + c + e] = q[e]; }
  }
  fold_pixel_lanes(s1, s2, w.lanes, width);
  if (p.dgamma || p.dbeta) {
    float* cp = p.cpart + ((size_t)b * p.strips + strip) * 2 * p.C;
    for (int c = threadIdx.x; c < p.C; c += (int)blockDim.x) { cp[c] = s1[c]; cp[p.C + c] = s2[c]; }
  }
  const int tpg = threads_per_group(p.G), j = threadIdx.x & (tpg - 1);
  for (int g0 = 0; g0 < p.G; g0 += (int)blockDim.x / tpg) {
    const int g = g0 + (int)threadIdx.x / tpg;
    float a = 0.f, q = 0.f;
    if (g < p.G)
      for (int c = j; c < p.cpg; c += tpg) {
        const float ga = p.gamma[g * p.cpg + c];
        a = fmaf(ga, s1[g * p.cpg + c], a);
        q = fmaf(ga, s2[g * p.cpg + c], q);
      }
    a = fold_lanes(a, tpg);
    q = fold_lanes(q, tpg);
    if (g < p.G && j == 0) {
      float* dst = p.part + (((size_t)b * p.strips + strip) * p.G + g) * 2;
      dst[0] = a; dst[1] = q;
    }
  }
}

// dgamma / dbeta: sum of `rows` rows [2][C] of channel sums; a block takes 16 channels x 16 row lanes.  In double: a lane adds
// up to 4096 rows one after the other (65535 samples of a slice each; in fp32 their rounding was 9 steps of dbeta).
constexpr int FOLD_LDS = 2 * 256 * 8;
__device__ __forceinline__ void fold_channels(const GnaParams& p, int block, int64_t rows, double* red) {
  const int cl = threadIdx.x & 15, rl = (threadIdx.x >> 4) & 15, c = block * 16 + cl;
  double a = 0.0, q = 0.0;
  if (threadIdx.x < 256 && c < p.C)
    for (int64_t r = rl; r < rows; r += 16) { a += (double)p.cpart[r * 2 * p.C + c]; q += (double)p.cpart[r * 2 * p.C + p.C + c]; }
  if (threadIdx.x < 256) { red[rl * 16 + cl] = a; red[256 + rl * 16 + cl] = q; }
  __syncthreads();
  if (threadIdx.x < 16 && c < p.C) {
    a = 0.0; q = 0.0;
#pragma unroll
    for (int r = 0; r < 16; ++r) { a += red[r * 16 + cl]; q += red[256 + r * 16 + cl]; }
    if (p.dbeta) p.dbeta[c] = (float)a;
    if (p.dgamma) p.dgamma[c] = (float)q;
  }
}
__global__ __launch_bounds__(256) void gna_fold_channels_kernel(GnaParams p, int64_t rows) {
  __shared__ double red[FOLD_LDS / 8];
  fold_channels(p, (int)blockIdx.x, rows, red);
}

// backward, second launch: dx; the blocks behind the strips' fold dgamma and dbeta
template <typename T, int ACT, bool DROP, bool WHOLE>
__global__ __launch_bounds__(1024) void gna_grad_apply_kernel(GnaParams p) {
  constexpr int WALK_BWD = Depth<T>::BWD;
  const int act = ACT < 0 ? p.act : ACT;
  extern __shared__ __align__(16) char smem[];
  if ((int)blockIdx.x >= p.apply_blocks) {
    if (blockIdx.y == 0)
      fold_channels(p, (int)blockIdx.x - p.apply_blocks, (int64_t)p.B * p.strips, reinterpret_cast<double*>(smem));
    return;
  }
  float* s_a = reinterpret_cast<float*>(smem);
  float* s_q = s_a + p.G;
  const int strip = blockIdx.x, b = blockIdx.y;
  const Walk w = walk_of(p, strip, b);
  typedef Cols<T, WHOLE> C;
  typename C::Raw rx[WALK_BWD], rd[WALK_BWD];
  const int c = w.cg * 8;
  const C x(p.x0, p.x1, p.c0, p.c1, c, w.row0), dy(p.dy, p.dy, p.C, 0, c, w.row0);
  if (w.live) {
    fetch(x, w, w.pl, rx);
    fetch(dy, w, w.pl, rd);
  }
  fold_strips(p, b, [](int, double, float2 v, double& a, double& q) { a += (double)v.x; q += (double)v.y; },
              [&](int g, double, double a, double q) {
    const double n = (double)p.HW * (double)p.cpg;
    s_a[g] = (float)(a / n); s_q[g] = (float)(q / n);
  });
  __syncthreads();
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  if (w.live) {
    const C dx(p.out0, p.out1, p.c0, p.c1, c, w.row0);
    // dx = rstd (h - a - xh q) = sc du - (rstd a + (x - mean) rstd^2 q)
    float mn[8], sc[8], bt[8], ka[8], kq[8];
    load_params(p.gamma, c, p.C, sc);
    load_params(p.beta, c, p.C, bt);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int g = (int)div_by((unsigned)(c + e < p.C ? c + e : p.C - 1), p.div_cpg);
      const float* st = p.stats + ((size_t)b * p.G + g) * 2;
      const float rs = st[1];
      mn[e] = st[0]; sc[e] *= rs;
      ka[e] = rs * s_a[g]; kq[e] = rs * rs * s_q[g];
    }
    const float ds = DROP ? p.drop.scale : 1.f;
    for (int px = w.pl; px < w.count; px += WALK_BWD * w.lanes) {
      typename C::Raw nx[WALK_BWD], nd[WALK_BWD];
#pragma unroll
      for (int u = 0; u < WALK_BWD; ++u) { nx[u] = rx[u]; nd[u] = rd[u]; }
      if (px + WALK_BWD * w.lanes < w.count) {
        fetch(x, w, px + WALK_BWD * w.lanes, rx);
        fetch(dy, w, px + WALK_BWD * w.lanes, rd);
      }
#pragma unroll
      for (int u = 0; u < WALK_BWD; ++u) {
        if (px + u * w.lanes >= w.count) break;
        const int64_t row = w.row0 + px + u * w.lanes;
        float v[8], d[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = to_f32<T>(nd[u][e]);
          d[e] = to_f32<T>(nx[u][e]) - mn[e];
          z[e] = fmaf(d[e], sc[e], bt[e]);
        }
        if (DROP) drop8(v, philox8(k0, k1, (unsigned)w.cg, (uint64_t)row, p.drop.offset), p.drop.thr, ds);
        act_grad_n<T>(z, v, act);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(sc[e], v[e], -fmaf(d[e], kq[e], ka[e]));
        dx.store(px + u * w.lanes, v);
      }
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------
struct GnaPlan {
  int slice;                    // 1: one workgroup per (sample, group)
  int w;                        // ... columns per access
  int lds;
  int threads, strips; int64_t px_per_strip;
  size_t part, cpart, total;    // workspace offsets
};
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

GnaPlan gna_plan(int B, int64_t HW, int c0, int c1, int G, int dtype, int backward) {
  GnaPlan pl = {};
  const int C = c0 + c1, cpg = C / G;
  const size_t esz = sdmi_dtype_size(dtype);
  const size_t per = backward ? esz + 4 : esz;
  pl.w = 1;
  for (int w = 8; w > 1; w >>= 1)
    if (cpg % w == 0 && c0 % w == 0) { pl.w = w; break; }
  // beyond 8192 accesses a slice keeps its workgroup longer than two launches over strips take (bf16, us forward:
  // 3x37x53x480, 15 channels a group one by one, 23 against 14; 16x32x32x960 in pairs 27 against 25; but 16x32x32x640 in
  // fours 17 against 23)
  if (HW * (cpg / pl.w) <= 8192 && (size_t)HW * cpg * per <= 60 * 1024) {
    pl.slice = 1;
    pl.lds = (int)((size_t)HW * cpg * per);
    pl.cpart = 0;
    pl.total = backward && B > 1 ? up256((size_t)B * 2 * C * 4) : 0;
    return pl;
  }
  // About 1024 waves' worth of threads on the chip at a time (128 registers each): 512 blocks of 512, every pixel lane at
  // least four pixels.  Every block of the second launch folds its sample's strips, so where few samples would get more
  // than 128 strips each, and where a row alone takes half a block, it is 256 blocks of 1024.  Forward + backward, bf16,
  // us: 16x64x64x320 80 (84 with the large blocks), 2x64x64x320 32 (42), 1x256x256x256 73 (90 with the small ones),
  // 1x40x30x2560 45 (56).  A lane adds at most 512 values one after the other.
  const int ncg = (C + 7) / 8;
  int lanes;
  int64_t strips;
  for (pl.threads = 512;; pl.threads = 1024) {
    lanes = ncg <= pl.threads ? pl.threads / ncg : 1;      // (a block of 512 is given up below if that is too few)
    const int64_t by_work = (HW + 4 * lanes - 1) / (4 * lanes);
    strips = ((1 << 18) / pl.threads + B - 1) / B;
    if (strips > by_work) strips = by_work;
    if (pl.threads == 1024 || (strips <= 128 && ncg <= 256)) break;
  }
  const int64_t by_sum = (HW + 512 * lanes - 1) / (512 * lanes);
  if (strips < by_sum) strips = by_sum;
  if (strips < 1) strips = 1;
  pl.px_per_strip = (HW + strips - 1) / strips;
  pl.px_per_strip = (pl.px_per_strip + 4 * lanes - 1) / (4 * lanes) * (4 * lanes);      // whole walks of every lane
  pl.strips = (int)((HW + pl.px_per_strip - 1) / pl.px_per_strip);
  pl.lds = 2 * lanes * ncg * 8 * 4;
  pl.part = 0;
  pl.cpart = up256((size_t)B * pl.strips * G * 2 * 4);
  pl.total = pl.cpart + (backward ? up256((size_t)B * pl.strips * 2 * C * 4) : 0);
  return pl;
}

int gna_check(const GroupNormActArgs& a, const char* who) {
  SDMI_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "%s: bad dtype %d", who, a.dtype);
  SDMI_REQUIRE(a.B >= 0 && a.HW >= 0 && a.c0 > 0 && a.c1 >= 0, "%s: bad size", who);
  const int64_t C = (int64_t)a.c0 + a.c1;
  SDMI_REQUIRE(C <= GNA_MAX_C, "%s: %lld channels, at most %d are supported", who, (long long)C, GNA_MAX_C);
  SDMI_REQUIRE(a.groups > 0 && C % a.groups == 0, "%s: %lld channels do not split into %d groups", who, (long long)C, a.groups);
  SDMI_REQUIRE(a.eps >= 0.f, "%s: negative eps", who);
  SDMI_REQUIRE(a.act >= 0 && a.act < ACT_COUNT, "%s: unknown activation %d", who, a.act);
  SDMI_REQUIRE(a.HW < ((int64_t)1 << 38), "%s: %lld pixels a sample are too many", who, (long long)a.HW);
  SDMI_REQUIRE(a.B <= 65535, "%s: batch %d is beyond 65535", who, a.B);
  return SDMI_OK;
}

GnaParams gna_params(const GroupNormActArgs& a, const GnaPlan& pl, const DropArgs& drop) {
  GnaParams p = {};
  p.x0 = a.x0; p.x1 = a.c1 ? a.x1 : nullptr; p.dy = a.dy;
  p.c0 = a.c0; p.c1 = a.c1; p.C = a.c0 + a.c1; p.G = a.groups; p.cpg = p.C / a.groups; p.B = a.B; p.HW = a.HW;
  p.div_cpg = fast_div((unsigned)(pl.slice ? p.cpg / pl.w : p.cpg));
  p.eps = a.eps; p.gamma = a.gamma; p.beta = a.beta; p.act = a.act; p.drop = drop; p.stats = a.stats;
  p.strips = pl.strips; p.px_per_strip = pl.px_per_strip;
  p.part = (float*)((char*)a.workspace + pl.part); p.cpart = (float*)((char*)a.workspace + pl.cpart);
  p.dgamma = a.dgamma; p.dbeta = a.dbeta;
  return p;
}

int slice_threads(const GnaPlan& pl, const GnaParams& p) {
  const int64_t nv = p.HW * (p.cpg / pl.w);
  int t = 64;
  while (t < 1024 && t * 2 < nv) t <<= 1;
  return t;
}

dim3 slice_grid(const GnaParams& p) {
  const unsigned total = (unsigned)p.B * (unsigned)p.G;
  return total <= SLICES_X ? dim3(total) : dim3(SLICES_X, (total + SLICES_X - 1) / SLICES_X);
}

// the kernels over strips with SiLU (others by a branch), dropout and whole column groups compiled in
#define GNA_LAUNCH(K, A, D, W, GRID, LDS) hipLaunchKernelGGL((K<T, A, D, W>), GRID, dim3(pl.threads), LDS, s, p)
#define GNA_VARIANTS_W(K, W, GRID, LDS)                                   \
  {                                                                       \
    if (p.drop.thr) {                                                     \
      if (p.act == ACT_SILU) GNA_LAUNCH(K, ACT_SILU, true, W, GRID, LDS); \
      else GNA_LAUNCH(K, -1, true, W, GRID, LDS);                         \
    } else {                                                              \
      if (p.act == ACT_SILU) GNA_LAUNCH(K, ACT_SILU, false, W, GRID, LDS);\
      else GNA_LAUNCH(K, -1, false, W, GRID, LDS);                        \
    }                                                                     \
  }
#define GNA_VARIANTS(K, GRID, LDS)                 \
  {                                                \
    if (whole) GNA_VARIANTS_W(K, true, GRID, LDS)  \
    else GNA_VARIANTS_W(K, false, GRID, LDS)       \
  }
// whole groups of eight columns in each source, and strips within 2 GiB (offsets of 32 bits)
bool gna_whole(const GnaParams& p) {
  return p.c0 % 8 == 0 && p.c1 % 8 == 0 && p.px_per_strip * (int64_t)p.C * 4 < ((int64_t)1 << 31);
}

template <typename T>
int gna_fwd(const GroupNormActArgs& a, const GnaPlan& pl, const DropArgs& drop, hipStream_t s) {
  GnaParams p = gna_params(a, pl, drop);
  p.out0 = a.out;
  char label[64] = "";
  if (prof_on()) snprintf(label, sizeof(label), "gn_act B%d HW%lld C%d", p.B, (long long)p.HW, p.C);
  ProfScope prof(PROF_GROUPNORM, s, 0.0, 2.0 * p.B * (double)p.HW * p.C * sizeof(T), label);
  if (pl.slice) {
    const dim3 grid = slice_grid(p), block(slice_threads(pl, p));
    if (pl.w == 8) hipLaunchKernelGGL((gna_slice_fwd_kernel<T, 8>), grid, block, pl.lds, s, p);
    else if (pl.w == 4) hipLaunchKernelGGL((gna_slice_fwd_kernel<T, 4>), grid, block, pl.lds, s, p);
    else if (pl.w == 2) hipLaunchKernelGGL((gna_slice_fwd_kernel<T, 2>), grid, block, pl.lds, s, p);
    else hipLaunchKernelGGL((gna_slice_fwd_kernel<T, 1>), grid, block, pl.lds, s, p);
  } else {
    const dim3 grid(pl.strips, p.B);
    const bool whole = gna_whole(p);
    if (whole) hipLaunchKernelGGL((gna_stats_kernel<T, true>), grid, dim3(pl.threads), pl.lds, s, p);
    else hipLaunchKernelGGL((gna_stats_kernel<T, false>), grid, dim3(pl.threads), pl.lds, s, p);
    GNA_VARIANTS(gna_apply_kernel, grid, 2 * p.G * 4)
  }
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

template <typename T>
int gna_bwd(const GroupNormActArgs& a, const GnaPlan& pl, const DropArgs& drop, hipStream_t s) {
  GnaParams p = gna_params(a, pl, drop);
  p.out0 = a.dx0; p.out1 = a.dx1;
  char label[64] = "";
  if (prof_on()) snprintf(label, sizeof(label), "gn_act bwd B%d HW%lld C%d", p.B, (long long)p.HW, p.C);
  ProfScope prof(PROF_GROUPNORM, s, 0.0, 3.0 * p.B * (double)p.HW * p.C * sizeof(T), label);
  const bool weights = p.dgamma || p.dbeta;
  const unsigned fold_blocks = weights ? (unsigned)(p.C + 15) / 16 : 0;
  if (pl.slice) {
    const dim3 grid = slice_grid(p), block(slice_threads(pl, p));
    if (pl.w == 8) hipLaunchKernelGGL((gna_slice_bwd_kernel<T, 8>), grid, block, pl.lds, s, p);
    else if (pl.w == 4) hipLaunchKernelGGL((gna_slice_bwd_kernel<T, 4>), grid, block, pl.lds, s, p);
    else if (pl.w == 2) hipLaunchKernelGGL((gna_slice_bwd_kernel<T, 2>), grid, block, pl.lds, s, p);
    else hipLaunchKernelGGL((gna_slice_bwd_kernel<T, 1>), grid, block, pl.lds, s, p);
    if (weights && p.B > 1) hipLaunchKernelGGL(gna_fold_channels_kernel, dim3(fold_blocks), dim3(256), 0, s, p, (int64_t)p.B);
  } else {
    const bool whole = gna_whole(p);
    GNA_VARIANTS(gna_grad_sums_kernel, dim3(pl.strips, p.B), pl.lds)
    p.apply_blocks = (a.dx0 || a.dx1) ? pl.strips : 0;
    const int lds = 2 * p.G * 4 > FOLD_LDS ? 2 * p.G * 4 : FOLD_LDS;
    if (p.apply_blocks + fold_blocks) GNA_VARIANTS(gna_grad_apply_kernel, dim3(p.apply_blocks + fold_blocks, p.B), lds)
  }
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

}  // namespace

int64_t groupnorm_act_workspace_bytes(int batch, int64_t hw, int c0, int c1, int groups, int dtype, int backward) {
  if (batch <= 0 || hw <= 0 || c0 <= 0 || c1 < 0 || groups <= 0 || (c0 + c1) % groups) return 0;
  return (int64_t)gna_plan(batch, hw, c0, c1, groups, dtype, backward).total;
}

int groupnorm_act(const GroupNormActArgs& a, hipStream_t stream) {
  SDMI_TRY(gna_check(a, "groupnorm_act"));
  DropArgs drop;
  SDMI_TRY(drop_args(&drop, a.p, a.seed, a.seed_dev, a.offset, "groupnorm_act"));
  if (a.B == 0 || a.HW == 0) return SDMI_OK;
  SDMI_REQUIRE(a.x0 && (a.x1 || !a.c1) && a.gamma && a.beta && a.out && a.stats, "groupnorm_act: null pointer");
  const GnaPlan pl = gna_plan(a.B, a.HW, a.c0, a.c1, a.groups, a.dtype, 0);
  SDMI_REQUIRE(pl.total == 0 || a.workspace, "groupnorm_act: this size needs a workspace of %lld bytes", (long long)pl.total);
  SDMI_DISPATCH_DTYPE(a.dtype, T, return gna_fwd<T>(a, pl, drop, stream));
  return SDMI_OK;
}

int groupnorm_act_backward(const GroupNormActArgs& a, hipStream_t stream) {
  SDMI_TRY(gna_check(a, "groupnorm_act_backward"));
  DropArgs drop;
  SDMI_TRY(drop_args(&drop, a.p, a.seed, a.seed_dev, a.offset, "groupnorm_act_backward"));
  if (!a.dx0 && !a.dx1 && !a.dgamma && !a.dbeta) return SDMI_OK;
  if (a.B == 0 || a.HW == 0) {
    GnaPlan pl = {};
    GnaParams p = gna_params(a, pl, drop);
    if (p.dgamma || p.dbeta) {
      hipLaunchKernelGGL(gna_fold_channels_kernel, dim3((p.C + 15) / 16), dim3(256), 0, stream, p, (int64_t)0);
      SDMI_CHECK_HIP(hipGetLastError());
    }
    return SDMI_OK;
  }
  SDMI_REQUIRE(a.dy && a.x0 && (a.x1 || !a.c1) && a.gamma && a.beta && a.stats, "groupnorm_act_backward: null pointer");
  SDMI_REQUIRE(!a.c1 || (a.dx0 != nullptr) == (a.dx1 != nullptr), "groupnorm_act_backward: dx of both sources or of neither");
  const GnaPlan pl = gna_plan(a.B, a.HW, a.c0, a.c1, a.groups, a.dtype, 1);
  SDMI_REQUIRE(pl.total == 0 || a.workspace, "groupnorm_act_backward: this size needs a workspace of %lld bytes",
               (long long)pl.total);
  SDMI_DISPATCH_DTYPE(a.dtype, T, return gna_bwd<T>(a, pl, drop, stream));
  return SDMI_OK;
}
