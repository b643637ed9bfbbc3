// Linear layer with its epilogue, and its gradients:
//   z = x W^T + b          y = [resid +] drop(act(z))
//   dz = drop(dy) act'(z)  dx = dz W       dW = dz^T x       db = column sums of dz
// All three products are one kernel, out[m][n] = sum_k Q(m, k) P(n, k), whose operands lie either with the
// contraction contiguous ("rows") or with the output index contiguous ("columns"):
//   forward  Q = x  rows,     P = W  rows
//   dx       Q = dz rows,     P = W  columns   (contraction over the layer's outputs)
//   dW       Q = dz columns,  P = x  columns   (contraction over the tokens, split over workgroups)
#include "act_drop.h"
#include "ops.h"
#include <stdio.h>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// ---- fragments -------------------------------------------------------------------------------------
// One fragment = 16 bytes per lane: lane l holds row l % 16 and the contraction indices of chunk l / 16 (8 halves, or
// 4 floats that four fp32 MFMA steps take one after the other; both operands use the same order, so it cancels out).
template <typename T> struct Frag;
template <> struct Frag<half_t> { typedef half_t type __attribute__((ext_vector_type(8))); };
template <> struct Frag<bf16_t> { typedef bf16_t type __attribute__((ext_vector_type(8))); };
template <> struct Frag<float>  { typedef float  type __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ f32x4 mma(Frag<half_t>::type a, Frag<half_t>::type b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Frag<bf16_t>::type a, Frag<bf16_t>::type b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(Frag<float>::type a, Frag<float>::type b, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
  return c;
}

// ---- epilogue --------------------------------------------------------------------------------------
struct Epilogue {
  const float* bias;            // [N] or null
  const void* resid; int64_t ldr;
  void* out; int64_t ldo;
  float* preact;                // [M][N] fp32 or null: z, for the backward pass
  int act;
  DropArgs drop;
  int64_t M; int N;
};

// columns n .. n + 7 of row m (n a multiple of 8; the row's last group may be short)
template <typename T>
__device__ __forceinline__ void finish8(const Epilogue& e, unsigned k0, unsigned k1, int64_t m, int n, float (&v)[8]) {
  const int cnt = e.N - n;
  if (e.bias) {
    float b[8];
    load8<float>(e.bias + n, cnt, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
  }
  if (e.preact) store8<float>(e.preact + m * e.N + n, cnt, v);
  if (e.act != ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_f<T>(v[i], e.act);
  }
  if (e.drop.thr) drop8(v, philox8(k0, k1, (unsigned)n >> 3, (uint64_t)m, e.drop.offset), e.drop.thr, e.drop.scale);
  if (e.resid) {
    float r[8];
    load8<T>((const T*)e.resid + m * e.ldr + n, cnt, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store8<T>((T*)e.out + m * e.ldo + n, cnt, v);
}

// ---- the product -----------------------------------------------------------------------------------
struct GemmParams {
  const char* q; const char* p;      // operands
  int64_t ldq, ldp;                  // elements from one stored row to the next
  int64_t K, k_per_split;            // contraction; a split's share is a multiple of the K-tile
  unsigned tiles_n, tiles, splits;
  float* partial;                    // [splits][M][N] fp32, or null: the kernel finishes the rows itself
  Epilogue e;
};

__device__ const u32x4 g_zero16 = {0, 0, 0, 0};      // contraction indices beyond the end are read here

__device__ __forceinline__ void glds16(const char* src, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

// An operand's K-tile in LDS is 8 ROWS chunks of 16 bytes; the contraction is KT = 128 bytes deep.
//   rows:    [ROWS][8 chunks], chunk index XORed with the row's low bits
//   columns: [KT][ROWS elements], chunk index XORed with a function of the contraction index that puts the rows one
//            transposing read touches into different banks
// The XOR is applied to the address a lane reads from (LDS-DMA writes lane by lane), and undone where fragments are read.
template <typename T, int ROWS, bool COLS> struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T), KT = 8 * EPC, CPR = ROWS / EPC;
  __device__ static __forceinline__ int swz(int k) {
    if constexpr (!COLS) return k & 7;
    else if constexpr (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
    else if constexpr (ROWS >= 128) return ((k & 3) | ((k >> 1) & 4)) << 1;
    else return (((k >> 1) & 1) | (((k >> 3) & 1) << 1)) << 1;
  }
  // what chunk `pos` of the tile holds: stored row a (output row, or contraction index), chunk c of it
  __device__ static __forceinline__ void at(int pos, int& a, int& c) {
    if constexpr (!COLS) { a = pos >> 3; c = (pos & 7) ^ swz(a); }
    else { a = pos / CPR; c = (pos % CPR) ^ swz(a); }
  }
  // fragment of rows r0 .. r0 + 15 (a multiple of 16), k-step kk (of 2)
  __device__ static __forceinline__ typename Frag<T>::type frag(const char* lds, int r0, int kk, int lane) {
    typedef typename Frag<T>::type F;
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!COLS) {
      const int row = r0 + i;
      return *reinterpret_cast<const F*>(lds + row * 128 + (((kk * 4 + g) ^ swz(row)) << 4));
    } else if constexpr (sizeof(T) == 4) {
      F f;
      const int k = kk * 16 + g * 4, c = (r0 + i) >> 2;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *reinterpret_cast<const float*>(lds + (k + e) * (ROWS * 4) + ((c ^ swz(k)) << 4) + ((i & 3) << 2));
      return f;
    } else {
      // two transposing reads of 4 contraction indices each: in every group of 16 lanes, lanes 4 j + q point at
      // columns 4 q .. 4 q + 3 of index j, and lane i gets column i of the four indices
      const int c = (r0 >> 3) + ((i & 3) >> 1);
      u32x2 h[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int k = kk * 32 + g * 8 + t * 4 + (i >> 2);
        const char* a = lds + k * (ROWS * 2) + ((c ^ swz(k)) << 4) + ((i & 1) << 3);
        h[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4*)(a)));
      }
      const u32x4 w = {h[0].x, h[0].y, h[1].x, h[1].y};
      return __builtin_bit_cast(F, w);
    }
  }
};

// A workgroup of WQ x WP waves, each FQ x FP fragments; NST LDS stages.  VEC: rows are whole 16-byte chunks at
// 16-byte addresses and go to LDS by DMA; otherwise chunks are put together in registers, element by element where
// they end, and written to the other stage behind the products.
template <typename T, int WQ, int WP, int FQ, int FP, int NST, bool QC, bool PC, bool VEC>
__global__ __launch_bounds__(64 * WQ * WP) void linear_gemm_kernel(GemmParams p) {
  constexpr int NW = WQ * WP, NT = 64 * NW, BM = 16 * WQ * FQ, BN = 16 * WP * FP;
  typedef Tile<T, BM, QC> TQ;
  typedef Tile<T, BN, PC> TP;
  constexpr int EPC = TQ::EPC, KT = TQ::KT, SZ = (int)sizeof(T);
  constexpr int NQ = BM * 8 / NT, NP = BN * 8 / NT, STAGE = (BM + BN) * 128;
  static_assert(NQ * NT == BM * 8 && NP * NT == BN * 8, "chunks must divide over the threads");
  static_assert(VEC || NST == 2, "register staging writes the other of two stages");
  static_assert(FP % 2 == 0, "the epilogue joins pairs of column fragments");
  __shared__ __align__(16) char smem[NST * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

  // workgroup -> (split, tile): ids go round-robin over the 8 XCDs, so each XCD takes a contiguous run; column tiles
  // of one row block are neighbours and share its Q tile in the XCD's L2
  const unsigned total = p.tiles * p.splits, xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
  const unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
  const unsigned split = id / p.tiles, tile = id - split * p.tiles;
  const unsigned tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = (int)tn * BN;
  const int64_t kb = (int64_t)split * p.k_per_split;
  const int64_t ke = kb + p.k_per_split < p.K ? kb + p.k_per_split : p.K;
  const int nk = (int)((ke - kb + KT - 1) / KT);

  // per-thread chunk sources.  Output rows beyond the end repeat the last ones (their results are not stored).
  const char* src[NQ + NP];
  int kidx[NQ + NP];                 // contraction index of the chunk inside a K-tile
  int cnt[NQ + NP];                  // columns operand: elements of the chunk inside the matrix (register staging)
  const int64_t stepq = QC ? (int64_t)KT * p.ldq * SZ : 128, stepp = PC ? (int64_t)KT * p.ldp * SZ : 128;
#pragma unroll
  for (int i = 0; i < NQ + NP; ++i) {
    const bool isq = i < NQ;
    const int pos = ((isq ? i : i - NQ) * NW + wave) * 64 + lane;
    int a, c;
    if (isq) TQ::at(pos, a, c); else TP::at(pos, a, c);
    const bool cols = isq ? QC : PC;
    const char* base = isq ? p.q : p.p;
    const int64_t ld = isq ? p.ldq : p.ldp;
    const int64_t r0 = isq ? m0 : (int64_t)n0, R = isq ? p.e.M : (int64_t)p.e.N;
    if (!cols) {
      const int64_t row = r0 + a < R ? r0 + a : R - 1;
      kidx[i] = c * EPC; cnt[i] = EPC;
      src[i] = base + (row * ld + kb + c * EPC) * SZ;
    } else {
      int64_t col = r0 + c * EPC;
      kidx[i] = a;
      if (VEC) { if (col > R - EPC) col = R - EPC; cnt[i] = EPC; }
      else { const int64_t left = R - col; cnt[i] = left < 0 ? 0 : (left > EPC ? EPC : (int)left); }
      src[i] = base + ((kb + a) * ld + col) * SZ;
    }
  }

  u32x4 reg[VEC ? 1 : NQ + NP];
  auto stage_in = [&](int t) {       // K-tile t: DMA into its stage, or loads into registers
    const int64_t left = ke - kb - (int64_t)t * KT;
    if constexpr (VEC) {
      char* buf = smem + (t % NST) * STAGE + wave * 1024;
      const char* zero = reinterpret_cast<const char*>(&g_zero16);
      const bool full = left >= KT;
#pragma unroll
      for (int i = 0; i < NQ + NP; ++i) {
        const char* s = full || kidx[i] < left ? src[i] : zero;
        glds16(s, buf + i * (NW * 1024));
        src[i] += i < NQ ? stepq : stepp;
      }
    } else {
      typedef typename Frag<T>::type F;
      typedef F Fu __attribute__((aligned(sizeof(T))));
#pragma unroll
      for (int i = 0; i < NQ + NP; ++i) {
        const bool cols = i < NQ ? QC : PC;
        const int64_t kleft = left - kidx[i];
        const int n = kleft <= 0 ? 0 : (cols ? cnt[i] : (kleft < EPC ? (int)kleft : EPC));
        F f;
        if (n == EPC) {
          f = *reinterpret_cast<const Fu*>(src[i]);
        } else {
#pragma unroll
          for (int e = 0; e < EPC; ++e) f[e] = e < n ? reinterpret_cast<const T*>(src[i])[e] : (T)0.f;
        }
        reg[i] = __builtin_bit_cast(u32x4, f);
        src[i] += i < NQ ? stepq : stepp;
      }
    }
  };
  auto regs_to_lds = [&](int t) {
    if constexpr (!VEC) {
      char* buf = smem + (t % NST) * STAGE + wave * 1024 + lane * 16;
#pragma unroll
      for (int i = 0; i < NQ + NP; ++i) *reinterpret_cast<u32x4*>(buf + i * (NW * 1024)) = reg[i];
    }
  };

  const int wq = wave % WQ, wp = wave / WQ;
  f32x4 acc[FP][FQ];
#pragma unroll
  for (int i = 0; i < FP; ++i)
#pragma unroll
    for (int j = 0; j < FQ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

  auto compute = [&](int t) {
    const char* lq = smem + (t % NST) * STAGE;
    const char* lp = lq + BM * 128;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      typename Frag<T>::type fp[FP], fq[FQ];
#pragma unroll
      for (int i = 0; i < FP; ++i) fp[i] = TP::frag(lp, wp * (16 * FP) + i * 16, kk, lane);
#pragma unroll
      for (int j = 0; j < FQ; ++j) fq[j] = TQ::frag(lq, wq * (16 * FQ) + j * 16, kk, lane);
#pragma unroll
      for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j) acc[i][j] = mma(fp[i], fq[j], acc[i][j]);
    }
  };

  if constexpr (VEC) {
    // ring of NST stages, one barrier per K-tile: a wave waits for its own part of tile t (younger tiles stay in
    // flight) and for its reads of tile t - 1; behind the barrier the whole tile is there, and the stage of tile
    // t - 1 is free for tile t + NST - 1
    constexpr int PER = NQ + NP;
#pragma unroll
    for (int t = 0; t < NST - 1; ++t)
      if (t < nk) stage_in(t);
    for (int t = 0; t < nk; ++t) {
      const int younger = nk - 1 - t < NST - 2 ? nk - 1 - t : NST - 2;
      if (younger <= 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      else if (younger == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PER) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * PER) : "memory");
      __builtin_amdgcn_s_barrier();
      if (t + NST - 1 < nk) stage_in(t + NST - 1);
      compute(t);
    }
  } else {
    if (nk > 0) { stage_in(0); regs_to_lds(0); }
    for (int t = 0; t < nk; ++t) {
      __syncthreads();
      if (t + 1 < nk) stage_in(t + 1);
      compute(t);
      if (t + 1 < nk) regs_to_lds(t + 1);      // last read in iteration t - 1, before this iteration's barrier
    }
  }

  // acc[i][j]: lane l holds columns 4 (l / 16) .. + 3 of fragment i, row l % 16 of fragment j.  Swapping 16-lane rows
  // between two column fragments leaves every lane with 8 consecutive columns (one generator call, 16-byte stores).
  const int g = lane >> 4;
  unsigned k0 = 0, k1 = 0;
  if (p.e.drop.thr && !p.partial) drop_key(p.e.drop, k0, k1);
#pragma unroll
  for (int j = 0; j < FQ; ++j) {
    const int64_t m = m0 + wq * (16 * FQ) + j * 16 + (lane & 15);
#pragma unroll
    for (int i = 0; i < FP; i += 2) {
      const int n = n0 + wp * (16 * FP) + i * 16 + (g & 1) * 16 + (g >> 1) * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, (float)acc[i][j][e]),
                                                        __builtin_bit_cast(unsigned, (float)acc[i + 1][j][e]), false, false);
        v[e] = __builtin_bit_cast(float, (unsigned)s[0]);
        v[4 + e] = __builtin_bit_cast(float, (unsigned)s[1]);
      }
      if (m < p.e.M && n < p.e.N) {
        if (p.partial) store8<float>(p.partial + ((int64_t)split * p.e.M + m) * p.e.N + n, p.e.N - n, v);
        else finish8<T>(p.e, k0, k1, m, n, v);
      }
    }
  }
}

// ---- joins -----------------------------------------------------------------------------------------
// Sum of the splits in a fixed order, then the epilogue; the blocks behind the rows' fold the bias gradient's strips.
struct JoinParams {
  const float* partial; unsigned splits;
  unsigned rows_per_y; FastDiv groups;
  Epilogue e;
  const float* db_partial; int strips, db_n; float* db;
  unsigned join_blocks;
};

template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(JoinParams p) {
  if (blockIdx.x >= p.join_blocks) {
    if (blockIdx.y) return;
    const int n = (int)(blockIdx.x - p.join_blocks) * 256 + (int)threadIdx.x;
    if (n >= p.db_n) return;
    float s = 0.f;
    for (int i = 0; i < p.strips; ++i) s += p.db_partial[(size_t)i * p.db_n + n];
    p.db[n] = s;
    return;
  }
  const int64_t row_base = (int64_t)blockIdx.y * p.rows_per_y, left = p.e.M - row_base;
  const unsigned rows = left < (int64_t)p.rows_per_y ? (unsigned)left : p.rows_per_y;
  const unsigned i = blockIdx.x * 256u + threadIdx.x;
  if (i >= rows * p.groups.d) return;
  const unsigned r = div_by(i, p.groups);
  const int n = (int)(i - r * p.groups.d) * 8;
  const int64_t m = row_base + r;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  for (unsigned s = 0; s < p.splits; ++s) {
    float w[8];
    load8<float>(p.partial + ((int64_t)s * p.e.M + m) * p.e.N + n, p.e.N - n, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  unsigned k0 = 0, k1 = 0;
  if (p.e.drop.thr) drop_key(p.e.drop, k0, k1);
  finish8<T>(p.e, k0, k1, m, n, v);
}

// ---- dz = drop(dy) act'(z), and the strips' column sums ----------------------------------------------
struct DzParams {
  const void* dy; int64_t lddy;
  const float* preact;          // [M][N], null without an activation
  void* dz;                     // [M][N], null: only the sums are wanted
  float* db_partial;            // [strips][N] or null
  int64_t M, rows_per_strip;
  int N, act;
  DropArgs drop;
};

// A block takes 32 column groups (256 columns) x 8 row lanes of a strip: consecutive threads read consecutive columns.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzParams p) {
  __shared__ float red[8][32 * 8 + 4];
  const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int n = (int)(blockIdx.x * 32 + cg) * 8;
  const int cnt = p.N - n;
  const int64_t rb = (int64_t)blockIdx.y * p.rows_per_strip;
  const int64_t re = rb + p.rows_per_strip < p.M ? rb + p.rows_per_strip : p.M;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  if (cnt > 0) {
    for (int64_t m = rb + rl; m < re; m += 8) {
      float v[8];
      load8<T>((const T*)p.dy + m * p.lddy + n, cnt, v);
      if (p.drop.thr) drop8(v, philox8(k0, k1, (unsigned)n >> 3, (uint64_t)m, p.drop.offset), p.drop.thr, p.drop.scale);
      if (p.act != ACT_NONE) {
        float z[8];
        load8<float>(p.preact + m * p.N + n, cnt, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= act_grad<T>(z[e], p.act);
      }
      if (p.dz) store8<T>((T*)p.dz + m * p.N + n, cnt, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += v[e];
    }
  }
  if (!p.db_partial) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) red[rl][cg * 8 + e] = s[e];
  __syncthreads();
  const int col = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (col < p.N) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += red[r][threadIdx.x];
    p.db_partial[(size_t)blockIdx.y * p.N + col] = t;
  }
}

// ---- host ------------------------------------------------------------------------------------------
// Tile and split of a product.  A workgroup of the large tile does the most work per byte it loads; when there are too
// few tiles to fill the chip the contraction is split, in shares that are worth a launch.
struct Plan { int bm, bn; unsigned tiles_m, tiles_n, splits; int64_t k_per_split; };

Plan plan_product(int64_t M, int N, int64_t K, int esize) {
  Plan pl;
  const int kt = 128 / esize;
  auto tiles = [&](int b) { return ((M + b - 1) / b) * (int64_t)((N + b - 1) / b); };
  int b = tiles(128) >= 192 ? 128 : 64;
  if (M > 512 && N > 512 && K >= 4096) b = 128;
  pl.bm = pl.bn = b;
  pl.tiles_m = (unsigned)((M + b - 1) / b); pl.tiles_n = (unsigned)((N + b - 1) / b);
  const int64_t t = tiles(b), nkt = (K + kt - 1) / kt;
  int64_t s = t >= 256 ? 1 : 512 / t;
  if (s > nkt / 4) s = nkt / 4;
  if (s < 1) s = 1;
  const int64_t per = (nkt + s - 1) / s;
  pl.k_per_split = per * kt;
  pl.splits = (unsigned)(nkt ? (nkt + per - 1) / per : 1);
  if (pl.k_per_split == 0) pl.k_per_split = kt;
  return pl;
}
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
size_t partial_bytes(const Plan& pl, int64_t M, int N) { return pl.splits > 1 ? up256((size_t)pl.splits * M * N * 4) : 0; }

bool chunked(const void* p, int64_t ld, int64_t len, int esize) {      // rows are whole 16-byte chunks at 16-byte addresses
  return ((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0 && (len * esize) % 16 == 0;
}

template <typename T, bool QC, bool PC, bool VEC>
void launch_tiles(const GemmParams& g, const Plan& pl, hipStream_t stream) {
  const dim3 grid(g.tiles * g.splits);
  if (pl.bm == 128) hipLaunchKernelGGL((linear_gemm_kernel<T, 2, 2, 4, 4, 2, QC, PC, VEC>), grid, dim3(256), 0, stream, g);
  else hipLaunchKernelGGL((linear_gemm_kernel<T, 2, 2, 2, 2, 2, QC, PC, VEC>), grid, dim3(256), 0, stream, g);
}

// db_*: a bias gradient to fold in the join's launch (or in one of its own)
struct DbFold { const float* partial = nullptr; int strips = 0, n = 0; float* db = nullptr; };

template <typename T>
int launch_join(const float* partial, unsigned splits, const Epilogue& e, const DbFold& f, hipStream_t stream) {
  JoinParams j;
  j.partial = partial; j.splits = splits; j.e = e;
  j.db_partial = f.partial; j.strips = f.strips; j.db_n = f.n; j.db = f.db;
  const unsigned groups = (unsigned)(e.N + 7) / 8;
  j.groups = fast_div(groups ? groups : 1);
  const int64_t cap = 0x70000000u / j.groups.d, rows = partial ? e.M : 0;
  j.rows_per_y = (unsigned)(rows < cap ? rows : cap);
  const unsigned ny = rows ? (unsigned)((rows + j.rows_per_y - 1) / j.rows_per_y) : 1u;
  j.join_blocks = (unsigned)(((uint64_t)j.rows_per_y * groups + 255) / 256);
  if (!partial) j.join_blocks = 0;
  const unsigned db_blocks = f.db ? (unsigned)(f.n + 255) / 256 : 0;
  hipLaunchKernelGGL(linear_join_kernel<T>, dim3(j.join_blocks + db_blocks, ny), dim3(256), 0, stream, j);
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

// out[m][n] = epilogue(sum_k Q(m, k) P(n, k)); `fold` rides on the join if there is one (returns whether it did)
template <typename T, bool QC, bool PC>
int product(const void* q, int64_t ldq, const void* p, int64_t ldp, int64_t K, const Epilogue& e, float* partial,
            const DbFold& fold, bool* folded, hipStream_t stream) {
  const int sz = (int)sizeof(T);
  const Plan pl = plan_product(e.M, e.N, K, sz);
  GemmParams g;
  g.q = (const char*)q; g.p = (const char*)p; g.ldq = ldq; g.ldp = ldp; g.K = K; g.k_per_split = pl.k_per_split;
  g.tiles_n = pl.tiles_n; g.splits = pl.splits; g.e = e;
  const uint64_t total = (uint64_t)pl.tiles_m * pl.tiles_n * pl.splits;
  SDMI_REQUIRE(total < (1ull << 31), "linear_act: %lld x %d outputs are too many", (long long)e.M, e.N);
  g.tiles = pl.tiles_m * pl.tiles_n;
  g.partial = pl.splits > 1 ? partial : nullptr;
  const bool vec = chunked(q, ldq, QC ? e.M : K, sz) && chunked(p, ldp, PC ? e.N : K, sz);
  {
    char label[96];
    snprintf(label, sizeof(label), "linear M%lld N%d K%lld", (long long)e.M, e.N, (long long)K);
    ProfScope prof(PROF_OTHER, stream, 2.0 * e.M * (double)e.N * K, 0.0, label);
    if (vec) launch_tiles<T, QC, PC, true>(g, pl, stream);
    else launch_tiles<T, QC, PC, false>(g, pl, stream);
    SDMI_CHECK_HIP(hipGetLastError());
  }
  if (g.partial) {
    SDMI_TRY(launch_join<T>(g.partial, g.splits, e, fold, stream));
    if (folded) *folded = fold.db != nullptr;
  }
  return SDMI_OK;
}

struct BwdLayout { size_t dz, dbp, px, pw, total; int strips; int64_t rows_per_strip; bool need_dz; };
BwdLayout bwd_layout(int64_t M, int K, int N, int act, bool drop, int want, int esize) {
  BwdLayout w;
  size_t o = 0;
  w.need_dz = (act != ACT_NONE || drop) && (want & 3);
  w.dz = o; o += w.need_dz ? up256((size_t)M * N * esize) : 0;
  // strips of rows: about 1024 blocks in all, at least 32 rows each
  const int64_t cblocks = (N + 255) / 256;
  int64_t strips = (1024 + cblocks - 1) / (cblocks ? cblocks : 1);
  if (strips > (M + 31) / 32) strips = (M + 31) / 32;
  if (strips < 1) strips = 1;
  w.rows_per_strip = (M + strips - 1) / strips;
  w.strips = w.rows_per_strip ? (int)((M + w.rows_per_strip - 1) / w.rows_per_strip) : 0;
  w.dbp = o; o += (want & 4) ? up256((size_t)w.strips * N * 4) : 0;
  w.px = o; o += (want & 1) ? partial_bytes(plan_product(M, K, N, esize), M, K) : 0;
  w.pw = o; o += (want & 2) ? partial_bytes(plan_product(N, K, M, esize), N, K) : 0;
  w.total = o;
  return w;
}

Epilogue plain_out(void* out, int64_t M, int N) {
  Epilogue e = {};
  e.out = out; e.ldo = N; e.M = M; e.N = N;
  return e;
}

template <typename T>
int linear_bwd(const LinearActArgs& a, const DropArgs& drop, hipStream_t s) {
  const int want = (a.dx ? 1 : 0) | (a.dw ? 2 : 0) | (a.db ? 4 : 0);
  const BwdLayout w = bwd_layout(a.rows, a.k, a.n, a.act, drop.thr != 0, want, (int)sizeof(T));
  char* ws = (char*)a.workspace;
  const void* dz = a.dy;
  int64_t lddz = a.lddy;
  DbFold fold;
  if (a.rows > 0 && (w.need_dz || a.db)) {
    DzParams d;
    d.dy = a.dy; d.lddy = a.lddy; d.preact = a.act != ACT_NONE ? a.preact : nullptr;
    d.dz = w.need_dz ? ws + w.dz : nullptr;
    d.db_partial = a.db ? (float*)(ws + w.dbp) : nullptr;
    d.M = a.rows; d.rows_per_strip = w.rows_per_strip; d.N = a.n; d.act = a.act; d.drop = drop;
    char label[64];
    snprintf(label, sizeof(label), "linear dz %lldx%d", (long long)a.rows, a.n);
    ProfScope prof(PROF_OTHER, s, 0.0, 2.0 * a.rows * (double)a.n * sizeof(T), label);
    hipLaunchKernelGGL(linear_dz_kernel<T>, dim3((a.n + 255) / 256, w.strips), dim3(256), 0, s, d);
    SDMI_CHECK_HIP(hipGetLastError());
    if (w.need_dz) { dz = d.dz; lddz = a.n; }
  }
  if (a.db) { fold.partial = (const float*)(ws + w.dbp); fold.strips = a.rows > 0 ? w.strips : 0; fold.n = a.n; fold.db = a.db; }
  bool folded = false;
  if (a.dw)
    SDMI_TRY((product<T, true, true>(dz, lddz, a.x, a.ldx, a.rows, plain_out(a.dw, a.n, a.k), (float*)(ws + w.pw), fold,
                                     &folded, s)));
  if (a.dx && a.rows > 0)
    SDMI_TRY((product<T, false, true>(dz, lddz, a.w, a.ldw, a.n, plain_out(a.dx, a.rows, a.k), (float*)(ws + w.px),
                                      folded ? DbFold() : fold, folded ? nullptr : &folded, s)));
  if (a.db && !folded) SDMI_TRY(launch_join<T>(nullptr, 0, plain_out(nullptr, 0, 0), fold, s));
  return SDMI_OK;
}

int check_common(const LinearActArgs& a, const char* who) {
  SDMI_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "%s: bad dtype %d", who, a.dtype);
  SDMI_REQUIRE(a.rows >= 0 && a.k > 0 && a.n > 0, "%s: bad size (%lld rows, %d inputs, %d outputs)", who,
               (long long)a.rows, a.k, a.n);
  SDMI_REQUIRE(a.act >= 0 && a.act < ACT_COUNT, "%s: unknown activation %d", who, a.act);
  SDMI_REQUIRE(a.ldx >= 0 && a.ldw >= 0 && a.ldr >= 0 && a.lddy >= 0, "%s: negative row stride", who);
  return SDMI_OK;
}

}  // namespace

int64_t linear_act_workspace_bytes(int64_t rows, int k, int n, int dtype) {
  if (rows <= 0 || k <= 0 || n <= 0) return 0;
  return (int64_t)partial_bytes(plan_product(rows, n, k, (int)sdmi_dtype_size(dtype)), rows, n);
}
int64_t linear_act_backward_workspace_bytes(int64_t rows, int k, int n, int act, double p, int want, int dtype) {
  if (rows <= 0 || k <= 0 || n <= 0) return 0;
  return (int64_t)bwd_layout(rows, k, n, act, p > 0.0, want, (int)sdmi_dtype_size(dtype)).total;
}

int linear_act(const LinearActArgs& a, hipStream_t stream) {
  SDMI_TRY(check_common(a, "linear_act"));
  Epilogue e = {};
  SDMI_TRY(drop_args(&e.drop, a.p, a.seed, a.seed_dev, a.offset, "linear_act"));
  if (a.rows == 0) return SDMI_OK;
  SDMI_REQUIRE(a.x && a.w && a.out, "linear_act: null pointer");
  const int64_t need = linear_act_workspace_bytes(a.rows, a.k, a.n, a.dtype);
  SDMI_REQUIRE(need == 0 || a.workspace, "linear_act: this size needs a workspace of %lld bytes", (long long)need);
  e.bias = a.bias; e.resid = a.resid; e.ldr = a.ldr; e.out = a.out; e.ldo = a.n;
  e.preact = a.act != ACT_NONE ? a.preact : nullptr; e.act = a.act; e.M = a.rows; e.N = a.n;
  SDMI_DISPATCH_DTYPE(a.dtype, T, return (product<T, false, false>(a.x, a.ldx, a.w, a.ldw, a.k, e, (float*)a.workspace,
                                                                     DbFold(), nullptr, stream)));
  return SDMI_OK;
}

int linear_act_backward(const LinearActArgs& a, hipStream_t stream) {
  SDMI_TRY(check_common(a, "linear_act_backward"));
  DropArgs drop;
  SDMI_TRY(drop_args(&drop, a.p, a.seed, a.seed_dev, a.offset, "linear_act_backward"));
  const int want = (a.dx ? 1 : 0) | (a.dw ? 2 : 0) | (a.db ? 4 : 0);
  if (!want) return SDMI_OK;
  if (a.rows > 0) {
    SDMI_REQUIRE(a.dy && (a.x || !a.dw) && (a.w || !a.dx), "linear_act_backward: null pointer");
    SDMI_REQUIRE(a.preact || a.act == ACT_NONE, "linear_act_backward: the activation's gradient needs preact");
    const int64_t need = linear_act_backward_workspace_bytes(a.rows, a.k, a.n, a.act, a.p, want, a.dtype);
    SDMI_REQUIRE(need == 0 || a.workspace, "linear_act_backward: this size needs a workspace of %lld bytes", (long long)need);
  }
  SDMI_DISPATCH_DTYPE(a.dtype, T, return linear_bwd<T>(a, drop, stream));
  return SDMI_OK;
}
