// Linear layer with its epilogue, and its gradients:
//   z = x W^T + b          y = [resid +] drop(act(z))
//   dz = drop(dy) act'(z)  dx = dz W       dW = dz^T x       db = column sums of dz
// All three products are one kernel, out[m][n] = sum_k Q(m, k) P(n, k), whose operands lie either with the
// contraction contiguous ("rows") or with the output index contiguous ("columns"):
//   forward  Q = x  rows,     P = W  rows
//   dx       Q = dz rows,     P = W  columns   (contraction over the layer's outputs)
//   dW       Q = dz columns,  P = x  columns   (contraction over the tokens, split over workgroups)
// Bounds, MI355X: the matrix rate where the contraction is long (8192x4096x4096 fp16: forward 220 us = 1249 TFLOP/s, dx 233,
// dW 227; a plain library product 212), HBM where it is short (65536x320x320 bf16: forward with bias, dropout and residual
// 38 us for 126 MB, dx 25 and dW 31 + 6 us), latency where there is little of anything (308x768x768 bf16 forward 8 us).
// With an activation 16-bit dx and dW take dz in two parts and twice the products' time (4096x1280x5120 bf16: 103 + 13 and
// 114 + 12 us, joins of the splits behind the plus).
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
  float alpha;                  // the sums are scaled by it first (1, or a gradient's dropout scale)
  int act;
  DropArgs drop;
  int64_t M; int N;
};

// columns n .. n + 7 of row m (n a multiple of 8; the row's last group may be short); r: the residual's, if there is one
// TAIL: short groups may come
template <typename T, bool TAIL>
__device__ __forceinline__ void finish8(const Epilogue& e, unsigned k0, unsigned k1, int64_t m, int n, const float (&r)[8],
                                        float (&v)[8]) {
  const int cnt = TAIL ? e.N - n : 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= e.alpha;
  if (e.bias) {
    float b[8];
    load8<float>(e.bias + n, cnt, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += b[i];
  }
  if (e.preact) store8<float>(e.preact + m * e.N + n, cnt, v);
  act_n<T>(v, e.act);
  if (e.drop.thr) drop8(v, philox8(k0, k1, (unsigned)n >> 3, (uint64_t)m, e.drop.offset), e.drop.thr, e.drop.scale);
  if (e.resid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store8<T>((T*)e.out + m * e.ldo + n, cnt, v);
}

// ---- the product -----------------------------------------------------------------------------------
// Column sums of the bias gradient's strips; rides on the launch of a product, in blocks behind its own.
struct DbFold { const float* partial = nullptr; int strips = 0, n = 0; float* db = nullptr; };
constexpr int DB_COLS = 16;          // columns a block folds, by 16 lanes each
__device__ __forceinline__ void fold_bias_gradient(const DbFold& f, int block, float* red) {
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4, n = block * DB_COLS + cl;
  float s = 0.f;
  if (n < f.n && rl < 16) {
    const float* src = f.partial + n;
    int i = rl;
    for (; i + 112 < f.strips; i += 128) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = src[(size_t)(i + 16 * u) * f.n];
      s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    for (; i < f.strips; i += 16) s += src[(size_t)i * f.n];
  }
  if (rl < 16) red[rl * 16 + cl] = s;
  __syncthreads();
  if (rl == 0 && n < f.n) {
    s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += red[r * 16 + cl];
    f.db[n] = s;
  }
}
__global__ __launch_bounds__(256) void linear_db_kernel(DbFold f) {
  __shared__ float red[256];
  fold_bias_gradient(f, (int)blockIdx.x, red);
}

struct GemmParams {
  const char* q; const char* p;      // operands
  const char* q2; float q_scale;     // q2 not null: a second Q, multiplied with the same P and added to the first one's sums times
                                     // q_scale (the first are then the second's low parts, held larger by 1 / q_scale)
  int64_t ldq, ldp;                  // elements from one stored row to the next
  int64_t K, k_per_split;            // contraction; a split's share is a multiple of the K-tile
  unsigned tiles_n, tiles, splits;
  float* partial;                    // [splits][M][N] fp32, or null: the kernel finishes the rows itself
  DbFold fold;
  Epilogue e;
};

// LDS-DMA of 16 bytes a lane from a uniform base plus a 32-bit offset; an offset beyond the 2 GiB that the descriptor
// spans is out of its bounds and brings zeros (contraction indices beyond the end)
constexpr unsigned DMA_SPAN = 0x80000000u, DMA_ZERO = 0x80000000u;
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned off, char* lds_wave_base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds_wave_base, 16, (int)off, 0, 0, 0);
}

// An operand's K-tile in LDS is 8 ROWS chunks of 16 bytes; the contraction is KT = 128 bytes deep.
//   rows:    [ROWS][8 chunks], chunk index XORed with the row's low bits
//   columns: [KT][ROWS elements], chunk index XORed with a function of the contraction index that puts the rows one
//            transposing read touches into different banks
// The XOR is applied to the address a lane reads from (LDS-DMA writes lane by lane), and undone where fragments are read.
template <typename T, int ROWS, bool COLS> struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T), KT = 8 * EPC, CPR = ROWS / EPC;
  static_assert(ROWS % 64 == 0, "the XOR stays inside a stored row");
  __device__ static __forceinline__ int swz(int k) {
    if constexpr (!COLS) return k & 7;
    else if constexpr (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
    else if constexpr (ROWS % 128 == 0) return ((k & 3) | ((k >> 1) & 4)) << 1;
    else return (((k >> 1) & 1) | (((k >> 3) & 1) << 1)) << 1;      // rows an odd multiple of 128 bytes apart
  }
  // what chunk `pos` of the tile holds: stored row a (output row, or contraction index), chunk c of it
  __device__ static __forceinline__ void at(int pos, int& a, int& c) {
    if constexpr (!COLS) { a = pos >> 3; c = (pos & 7) ^ swz(a); }
    else { a = pos / CPR; c = (pos % CPR) ^ swz(a); }
  }
  // fragment dyn + i of sixteen rows, k-step kk (of 2); dyn is the wave's, i a constant, and they have no bit in common:
  // the chunk XOR then is one value per lane that constants are XORed to and added to
  __device__ static __forceinline__ typename Frag<T>::type frag(const char* lds, int dyn, int i, int kk, int lane) {
    typedef typename Frag<T>::type F;
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!COLS) {
      return *reinterpret_cast<const F*>(lds + (dyn * 16 + r) * 128 + (((kk * 4 + g) ^ (r & 7)) << 4) + i * 2048);
    } else if constexpr (sizeof(T) == 4) {
      F f;
      const int k = kk * 16 + g * 4, c = (dyn + i) * 4 + (r >> 2);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = *reinterpret_cast<const float*>(lds + (k + e) * (ROWS * 4) + ((c ^ swz(k)) << 4) + ((r & 3) << 2));
      return f;
    } else {
      // two transposing reads of 4 contraction indices each: in every group of 16 lanes, lanes 4 j + q point at
      // columns 4 q .. 4 q + 3 of index j, and lane r gets column r of the four indices
      constexpr int MASK = ROWS % 128 == 0 ? 7 : 3;            // fragments the XOR permutes among themselves
      const int k = g * 8 + (r >> 2);                          // swz(k) is that of every index read here
      const int lane_at = k * (ROWS * 2) + ((r & 3) << 3);
      const int seg = dyn ^ (swz(k) >> 1) ^ (i & MASK);
      const char* a = lds + lane_at + (seg << 5) + ((i & ~MASK) << 5) + kk * 32 * (ROWS * 2);
      u32x2 h[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        h[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                   (__attribute__((address_space(3))) s16x4*)(a + t * 4 * (ROWS * 2))));
      const u32x4 w = {h[0].x, h[0].y, h[1].x, h[1].y};
      return __builtin_bit_cast(F, w);
    }
  }
};

// Column fragment i of wave group wp: the wave's own run of FP, but for FP = 10 (no power of two) eight of a run and two
// behind all runs, so that the wave's part and the constant part of the index have no bit in common.
template <int FP, int WP> __device__ __forceinline__ int col_dyn(int wp, int i) {
  if constexpr (FP == 10) return i < 8 ? wp * 8 : WP * 8 + wp * 2; else return wp * FP;
}
template <int FP> __device__ __forceinline__ constexpr int col_const(int i) { return FP == 10 && i >= 8 ? i - 8 : i; }

// A workgroup of WQ x WP waves, each FQ x FP fragments; two LDS stages.  VEC: rows are whole 16-byte chunks at 16-byte
// addresses and go to LDS by DMA; otherwise chunks are put together in registers, element by element where they end,
// and written to the other stage behind the products.
// VEC also means whole groups of eight output columns.
// PAIR > 0 (the large tiles, one workgroup per CU): the wave groups wp = 0 and 1, one wave of each per SIMD, run the same
// program one segment apart, so that one group reads fragments while the other keeps the matrix cores busy; a k-step
// is PAIR segments of FP / PAIR column fragments.
constexpr int NST = 2;             // stages
template <int WQ, int WP, int FQ, int FP> constexpr int lds_bytes() { return NST * 16 * (WQ * FQ + WP * FP) * 128; }
template <typename T, int WQ, int WP, int FQ, int FP, bool QC, bool PC, bool VEC, int PAIR>
__device__ __forceinline__ void gemm_block(const GemmParams& p, const unsigned block, char* smem) {
  constexpr int NW = WQ * WP, NT = 64 * NW, BM = 16 * WQ * FQ, BN = 16 * WP * FP;
  typedef Tile<T, BM, QC> TQ;
  typedef Tile<T, BN, PC> TP;
  constexpr int EPC = TQ::EPC, KT = TQ::KT, SZ = (int)sizeof(T);
  constexpr int NQ = BM * 8 / NT, NP = BN * 8 / NT, STAGE = (BM + BN) * 128;
  static_assert(NQ * NT == BM * 8 && NP * NT == BN * 8, "chunks must divide over the threads");
  static_assert(!PAIR || (VEC && WP == 2), "two groups of waves, staged by DMA");
  static_assert(FP % 2 == 0, "the epilogue's column groups divide over the lanes");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

  // workgroup -> (split, tile): ids go round-robin over the 8 XCDs, so each XCD takes a contiguous run; column tiles
  // of one row block are neighbours and share its Q tile in the XCD's L2
  if (block >= p.tiles * p.splits) {
    fold_bias_gradient(p.fold, (int)(block - p.tiles * p.splits), reinterpret_cast<float*>(smem));
    return;
  }
  const unsigned total = p.tiles * p.splits, xcd = block & 7, q8 = total >> 3, r8 = total & 7;
  const unsigned id = xcd * q8 + (xcd < r8 ? xcd : r8) + (block >> 3);
  const unsigned split = id / p.tiles, tile = id - split * p.tiles;
  const unsigned tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = (int)tn * BN;
  const int64_t kb = (int64_t)split * p.k_per_split;
  const int64_t ke = kb + p.k_per_split < p.K ? kb + p.k_per_split : p.K;
  const int nk1 = (int)((ke - kb + KT - 1) / KT), nk = p.q2 ? 2 * nk1 : nk1;

  // Per-thread chunk sources: offsets from a uniform base that moves with the K-tile.  Output rows beyond the end repeat
  // the last ones (their results are not stored).  Chunk i of a thread lies i * NT chunks behind its first one.
  const int64_t startq = (QC ? kb * p.ldq + m0 : m0 * p.ldq + kb) * SZ;
  const int64_t startp = (PC ? kb * p.ldp + n0 : (int64_t)n0 * p.ldp + kb) * SZ;
  const char* baseq = p.q + startq;
  const char* basep = p.p + startp;
  const int64_t stepq = QC ? (int64_t)KT * p.ldq * SZ : 128, stepp = PC ? (int64_t)KT * p.ldp * SZ : 128;
  const int64_t leftq = p.e.M - m0, leftp = (int64_t)p.e.N - n0;      // output rows / columns from this tile on
  auto place = [&](int i, bool isq, int& a, int& c) {
    const int pos = (i * NW + wave) * 64 + lane;
    if (isq) TQ::at(pos, a, c); else TP::at(pos, a, c);
  };
  unsigned off[VEC ? NQ + NP : 1];
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < NQ + NP; ++i) {
      const bool isq = i < NQ, cols = isq ? QC : PC;
      const int64_t ld = isq ? p.ldq : p.ldp, left = isq ? leftq : leftp;
      int a, c;
      place(isq ? i : i - NQ, isq, a, c);
      if (!cols) off[i] = (unsigned)(((a < left ? a : left - 1) * ld + c * EPC) * SZ);
      else off[i] = (unsigned)((a * ld + (c * EPC + EPC <= left ? c * EPC : left - EPC)) * SZ);
    }
  }

  const T* src[VEC ? 1 : NQ + NP];   // register staging: any stride, so whole addresses
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < NQ + NP; ++i) {
      const bool isq = i < NQ, cols = isq ? QC : PC;
      const int64_t ld = isq ? p.ldq : p.ldp, left = isq ? leftq : leftp;
      int a, c;
      place(isq ? i : i - NQ, isq, a, c);
      src[i] = reinterpret_cast<const T*>(isq ? baseq : basep) + (cols || a < left ? a : left - 1) * ld + c * EPC;
    }
  }

  u32x4 reg[VEC ? 1 : NQ + NP];
  auto stage_in = [&](int t) {       // K-tile t: DMA into its stage, or loads into registers; called for t = 0, 1, 2, ...
    if (t == nk1) {                  // once more, with the second Q
      if constexpr (VEC) { baseq = p.q2 + startq; basep = p.p + startp; }
      else {
        const int64_t backq = (p.q2 - p.q) - nk1 * stepq, backp = -nk1 * stepp;
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) src[i] = reinterpret_cast<const T*>(reinterpret_cast<const char*>(src[i]) + (i < NQ ? backq : backp));
      }
    }
    const int64_t left = ke - kb - (int64_t)(t < nk1 ? t : t - nk1) * KT;
    if constexpr (VEC) {
      char* buf = smem + (t % NST) * STAGE + wave * 1024;
      const auto rq = __builtin_amdgcn_make_buffer_rsrc((void*)baseq, 0, DMA_SPAN, 0x00020000);
      const auto rp = __builtin_amdgcn_make_buffer_rsrc((void*)basep, 0, DMA_SPAN, 0x00020000);
      if (left >= KT) {
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) dma16(i < NQ ? rq : rp, off[i], buf + i * (NW * 1024));
      } else {
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) {
          const bool isq = i < NQ, cols = isq ? QC : PC;
          int a, c;
          place(isq ? i : i - NQ, isq, a, c);
          dma16(isq ? rq : rp, (cols ? a : c * EPC) < left ? off[i] : DMA_ZERO, buf + i * (NW * 1024));
        }
      }
    } else {
      typedef typename Frag<T>::type F;
      typedef F Fu __attribute__((aligned(sizeof(T))));
      if (left >= KT && (!QC || leftq >= BM) && (!PC || leftp >= BN)) {      // every chunk is whole
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) {
          reg[i] = __builtin_bit_cast(u32x4, (F)*reinterpret_cast<const Fu*>(src[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) {
          const bool cols = i < NQ ? QC : PC;
          int a, c;
          place(i < NQ ? i : i - NQ, i < NQ, a, c);
          // elements of the chunk that are there
          const int64_t have = cols ? (a < left ? (i < NQ ? leftq : leftp) - c * EPC : 0) : left - c * EPC;
          F f;
          if (have >= EPC) {
            f = *reinterpret_cast<const Fu*>(src[i]);
          } else {
#pragma unroll
            for (int e = 0; e < EPC; ++e) f[e] = e < have ? src[i][e] : (T)0.f;
          }
          reg[i] = __builtin_bit_cast(u32x4, f);
        }
      }
#pragma unroll
      for (int i = 0; i < NQ + NP; ++i) src[i] = reinterpret_cast<const T*>(reinterpret_cast<const char*>(src[i]) + (i < NQ ? stepq : stepp));
    }
    baseq += stepq;
    basep += stepp;
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
  auto begin_tile = [&](int t) {     // before the products of K-tile t: behind the first Q its sums are scaled
    if constexpr (PC) {              // (a forward product has one Q)
      if (t == nk1) {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
          for (int j = 0; j < FQ; ++j) acc[i][j] *= p.q_scale;
      }
    }
  };

  constexpr int PH = PAIR ? PAIR : 1, FPH = FP / PH;
  static_assert(FPH * PH == FP, "segments share the column fragments evenly");
  typename Frag<T>::type fp[FPH], fq[FQ];
  auto read_frags = [&](int t, int kk, int ph) {
    const char* lq = smem + (t % NST) * STAGE;
    const char* lp = lq + BM * 128;
#pragma unroll
    for (int i = 0; i < FPH; ++i) {
      const int f = ph * FPH + i;
      fp[i] = TP::frag(lp, col_dyn<FP, WP>(wp, f), col_const<FP>(f), kk, lane);
    }
    if (ph == 0) {
#pragma unroll
      for (int j = 0; j < FQ; ++j) fq[j] = TQ::frag(lq, wq * FQ, j, kk, lane);
    }
  };
  auto multiply = [&](int ph) {
#pragma unroll
    for (int i = 0; i < FPH; ++i)
#pragma unroll
      for (int j = 0; j < FQ; ++j) acc[ph * FPH + i][j] = mma(fp[i], fq[j], acc[ph * FPH + i][j]);
  };

  if constexpr (PAIR > 0) {
    // Between two barriers one group reads the fragments of a segment and the other multiplies; group 1 enters one
    // barrier late.  With I = 4 PH intervals to a K-tile, tile t is read in the intervals I t .. I t + I - 1; its stage
    // takes the DMA of tile t + 2 from interval I t + I on, and every wave waits for its own part of that before the
    // barrier that ends interval I t + 2 I - 1.
    auto barrier = [&]() {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };
    if (nk > 0) stage_in(0);
    if (nk > 1) {
      stage_in(1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NQ + NP) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    barrier();
    if (wp == 1) barrier();
    for (int t = 0; t < nk; ++t) {
      begin_tile(t);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int ph = 0; ph < PH; ++ph) {
          const bool last = kk == 1 && ph == PH - 1;
          read_frags(t, kk, ph);
          if (kk == 0 && ph == 0 && t >= 1 && t + 1 < nk) stage_in(t + 1);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (last && wp == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          barrier();
          __builtin_amdgcn_s_setprio(1);
          multiply(ph);
          __builtin_amdgcn_s_setprio(0);
          if (last && wp == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          barrier();
        }
    }
    if (wp == 0) barrier();
  } else if constexpr (VEC) {
    // one barrier per K-tile: a wave waits for its own part of tile t and for its reads of tile t - 1; behind the
    // barrier the whole tile is there, and the stage of tile t - 1 is free for tile t + 1
    if (nk > 0) stage_in(0);
    for (int t = 0; t < nk; ++t) {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      if (t + 1 < nk) stage_in(t + 1);
      begin_tile(t);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) { read_frags(t, kk, 0); multiply(0); }
    }
  } else {
    if (nk > 0) { stage_in(0); regs_to_lds(0); }
    for (int t = 0; t < nk; ++t) {
      __syncthreads();
      if (t + 1 < nk) stage_in(t + 1);
      begin_tile(t);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) { read_frags(t, kk, 0); multiply(0); }
      if (t + 1 < nk) regs_to_lds(t + 1);      // last read in iteration t - 1, before this iteration's barrier
    }
  }

  // acc[i][j]: lane l holds columns 4 (l / 16) .. + 3 of fragment i, row l % 16 of fragment j.  Each wave takes its tile
  // through LDS sixteen rows at a time, so that a lane ends up with eight consecutive columns (one generator call) and
  // neighbouring lanes with neighbouring columns (whole lines to memory).  The residual of the next sixteen rows is
  // on its way meanwhile, and goes through LDS too, so that the loop over a lane's items stays rolled: unrolled it
  // would be 20 copies of the epilogue.
  typedef typename Vec8u<T>::type V8;
  constexpr int PITCH = 16 * FP + 4, ITEMS = FP / 2, GPR = 2 * FP;      // floats; items per lane; column groups per row
  constexpr int STRIP = 16 * PITCH * 4, RES = 16 * 16 * FP * SZ;
  static_assert(NW * (STRIP + RES) <= NST * STAGE, "the strips reuse the stages");
  if constexpr (PAIR == 0) __syncthreads();      // (the groups' last barrier stands behind every read of the stages)
  float* strip = reinterpret_cast<float*>(smem + wave * (STRIP + RES));
  typedef T V8a __attribute__((ext_vector_type(8)));
  V8a* rstrip = reinterpret_cast<V8a*>(smem + wave * (STRIP + RES) + STRIP);
  const bool resid = p.e.resid && !p.partial;
  unsigned k0 = 0, k1 = 0;
  if (p.e.drop.thr && !p.partial) drop_key(p.e.drop, k0, k1);
  auto col_of = [&](int grp) {                   // first column of the wave's group of eight
    const int i = grp >> 1;
    return n0 + (col_dyn<FP, WP>(wp, i) + col_const<FP>(i)) * 16 + (grp & 1) * 8;
  };
  const int64_t mw0 = m0 + wq * (16 * FQ);
  V8 res[ITEMS];
  auto load_resid = [&](int j) {
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
      const int idx = q * 64 + lane, row = idx / GPR, n = col_of(idx - row * GPR);
      const int64_t m = mw0 + j * 16 + row;
      if (m < p.e.M && n < p.e.N) {
        const T* r = (const T*)p.e.resid + m * p.e.ldr + n;
        if (VEC || n + 8 <= p.e.N) res[q] = *reinterpret_cast<const V8*>(r);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) res[q][e] = n + e < p.e.N ? r[e] : (T)0.f;
        }
      }
    }
  };
  auto wave_sync = [&]() {                        // the wave's own LDS writes before its reads, and the other way round
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  if (resid) load_resid(0);
#pragma unroll
  for (int j = 0; j < FQ; ++j) {
#pragma unroll
    for (int i = 0; i < FP; ++i)
      *reinterpret_cast<f32x4*>(strip + (lane & 15) * PITCH + i * 16 + (lane >> 4) * 4) = acc[i][j];
    if (resid) {
#pragma unroll
      for (int q = 0; q < ITEMS; ++q) rstrip[q * 64 + lane] = res[q];
      if (j + 1 < FQ) load_resid(j + 1);
    }
    wave_sync();
#pragma unroll 1
    for (int q = 0; q < ITEMS; ++q) {
      const int idx = q * 64 + lane, row = idx / GPR, grp = idx - row * GPR;
      const int64_t m = mw0 + j * 16 + row;
      const int n = col_of(grp);
      float v[8], r[8];
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(strip + row * PITCH + grp * 8);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(strip + row * PITCH + grp * 8 + 4);
      if (resid) {
        const V8a rr = rstrip[idx];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = to_f32<T>(rr[e]);
      }
      if (m < p.e.M && n < p.e.N) {
        if (p.partial) store8<float>(p.partial + ((int64_t)split * p.e.M + m) * p.e.N + n, VEC ? 8 : p.e.N - n, v);
        else finish8<T, !VEC>(p.e, k0, k1, m, n, r, v);
      }
    }
    wave_sync();
  }
}
template <typename T, int WQ, int WP, int FQ, int FP, bool QC, bool PC, bool VEC, int PAIR>
__global__ __launch_bounds__(64 * WQ * WP) void linear_gemm_kernel(GemmParams p) {
  __shared__ __align__(16) char smem[lds_bytes<WQ, WP, FQ, FP>()];
  gemm_block<T, WQ, WP, FQ, FP, QC, PC, VEC, PAIR>(p, blockIdx.x, smem);
}
// dW and dx in one launch: products that leave CUs idle one after the other share them.  us, replayed, apart / together:
// 308x768x768 bf16 13.4 / 9.2 (with an activation's dz in two parts 22.6 / 16.5), 406x256x384 fp16 11.2 / 6.4, 1003x517x259 fp32
// 28.1 / 23.6, 22932x128x2112 fp16 63 / 62 (218 / 211); over 300 sizes 1.33 times faster at the mean, 0.93 at worst
template <typename T, int FQ, int FP, bool VEC>
__global__ __launch_bounds__(256) void linear_grads_kernel(GemmParams w, GemmParams x) {
  __shared__ __align__(16) char smem[lds_bytes<2, 2, FQ, FP>()];
  const unsigned first = w.tiles * w.splits;
  if (blockIdx.x < first) gemm_block<T, 2, 2, FQ, FP, true, true, VEC, 0>(w, blockIdx.x, smem);
  else gemm_block<T, 2, 2, FQ, FP, false, true, VEC, 0>(x, blockIdx.x - first, smem);
}

// ---- few rows ----------------------------------------------------------------------------------------
// Forward for a handful of tokens: the weights pass through once and nothing is shared, so nothing goes through LDS on
// the way.  A workgroup takes 16 columns; its eight waves share the contraction in steps of one fragment, four steps' loads
// in flight each, and meet in LDS.  One launch, no workspace.
template <typename T, int FQ>
__global__ __launch_bounds__(512) void linear_few_kernel(GemmParams p) {
  typedef typename Frag<T>::type F;
  typedef F Fu __attribute__((aligned(sizeof(T))));
  constexpr int EPC = 16 / (int)sizeof(T), STEP = 4 * EPC, NW = 8, U = 4, PITCH = 20;
  __shared__ __align__(16) float red[NW][16 * FQ][PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, M = (int)p.e.M;
  const T* wrow = reinterpret_cast<const T*>(p.p) + (int64_t)(n0 + r < p.e.N ? n0 + r : p.e.N - 1) * p.ldp;
  const T* xrow[FQ];
#pragma unroll
  for (int j = 0; j < FQ; ++j) xrow[j] = reinterpret_cast<const T*>(p.q) + (int64_t)min(j * 16 + r, M - 1) * p.ldq;
  f32x4 acc[FQ];
#pragma unroll
  for (int j = 0; j < FQ; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  auto chunk = [&](const T* row, int64_t k) -> F {       // indices k .. k + EPC - 1, zeros beyond the end
    if (k + EPC <= p.K) return *reinterpret_cast<const Fu*>(row + k);
    F f;
#pragma unroll
    for (int e = 0; e < EPC; ++e) f[e] = k + e < p.K ? row[k + e] : (T)0.f;
    return f;
  };
  const int64_t whole = p.K - p.K % STEP;                // steps without an end in them
  int64_t k = (int64_t)wave * STEP + g * EPC;
  for (; k - g * EPC + (U - 1) * NW * STEP < whole; k += U * NW * STEP) {
    F w[U], x[U][FQ];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = *reinterpret_cast<const Fu*>(wrow + k + u * NW * STEP);
#pragma unroll
      for (int j = 0; j < FQ; ++j) x[u][j] = *reinterpret_cast<const Fu*>(xrow[j] + k + u * NW * STEP);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < FQ; ++j) acc[j] = mma(w[u], x[u][j], acc[j]);
  }
  for (; k - g * EPC < p.K; k += NW * STEP) {
    const F w = chunk(wrow, k);
#pragma unroll
    for (int j = 0; j < FQ; ++j) acc[j] = mma(w, chunk(xrow[j], k), acc[j]);
  }
#pragma unroll
  for (int j = 0; j < FQ; ++j) *reinterpret_cast<f32x4*>(&red[wave][j * 16 + r][g * 4]) = acc[j];
  __syncthreads();
  const int row = threadIdx.x >> 1, n = n0 + (threadIdx.x & 1) * 8;
  if (row >= M || n >= p.e.N) return;
  float v[8], res[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = 0.f;
#pragma unroll
    for (int s = 0; s < NW; ++s) v[e] += red[s][row][(threadIdx.x & 1) * 8 + e];
  }
  unsigned k0 = 0, k1 = 0;
  if (p.e.drop.thr) drop_key(p.e.drop, k0, k1);
  if (p.e.resid) load8<T>((const T*)p.e.resid + row * p.e.ldr + n, p.e.N - n, res);
  finish8<T, true>(p.e, k0, k1, row, n, res, v);
}
// where it beats the tiles (us, replayed, few / tiles): fp16 32x1280x1280 5.8 / 9.0, 16x2560x640 6.8 / 6.8,
// 8x5120x1280 9.6 / 8.0; fp32 2x1280x1280 5.8 / 8.6, 16x2560x640 11.3 / 9.3
bool few_rows(int64_t rows, int64_t k, int n, int esize) {
  return rows <= 32 && k * esize * (8 + rows) <= (128 << 10) && n <= (1 << 26);      // (a launch has less than 2^32 threads)
}

// ---- joins -----------------------------------------------------------------------------------------
// Sum of the splits in a fixed order, then the epilogue.  A group of eight columns is summed by LANES threads, each over
// every LANES-th split (four loads in flight), and finished by the first of them.  HBM, or latency where the outputs are
// few: 3 splits of 4096x1280 bf16 13 us (73 MB); 32 splits of 320x320 6 us (one thread a group: 19).
struct JoinParams {
  const float* partial; unsigned splits;
  unsigned rows_per_y; FastDiv groups;
  Epilogue e;
};

template <typename T, int LANES>
__global__ __launch_bounds__(256) void linear_join_kernel(JoinParams p) {
  __shared__ float red[LANES > 1 ? LANES - 1 : 1][256 / LANES][8];
  constexpr unsigned GROUPS = 256 / LANES;
  const int64_t row_base = (int64_t)blockIdx.y * p.rows_per_y, left = p.e.M - row_base;
  const unsigned rows = left < (int64_t)p.rows_per_y ? (unsigned)left : p.rows_per_y;
  const unsigned gl = threadIdx.x % GROUPS, sl = threadIdx.x / GROUPS;
  const unsigned i = blockIdx.x * GROUPS + gl;
  const bool live = i < rows * p.groups.d;
  const unsigned r = div_by(live ? i : 0, p.groups);
  const int n = (int)((live ? i : 0) - r * p.groups.d) * 8;
  const int64_t m = row_base + r;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (live) {
    const float* src = p.partial + m * p.e.N + n;
    const int64_t step = p.e.M * p.e.N;
    const int cnt = p.e.N - n;
    unsigned s = sl;
    for (; s + 3 * LANES < p.splits; s += 4 * LANES) {
      float w[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u) load8<float>(src + (s + u * LANES) * step, cnt, w[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += (w[0][e] + w[1][e]) + (w[2][e] + w[3][e]);
    }
    for (; s < p.splits; s += LANES) {
      float w[8];
      load8<float>(src + s * step, cnt, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
  }
  if constexpr (LANES > 1) {
    if (sl > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[sl - 1][gl][e] = v[e];
    }
    __syncthreads();
    if (sl > 0) return;
#pragma unroll
    for (int l = 0; l < LANES - 1; ++l)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += red[l][gl][e];
  }
  if (!live) return;
  unsigned k0 = 0, k1 = 0;
  if (p.e.drop.thr) drop_key(p.e.drop, k0, k1);
  float r8[8];
  if (p.e.resid) load8<T>((const T*)p.e.resid + m * p.e.ldr + n, p.e.N - n, r8);
  finish8<T, true>(p.e, k0, k1, m, n, r8, v);
}

// ---- dz = drop(dy) act'(z), and the strips' column sums ----------------------------------------------
// HBM (65536x320 bf16 without an activation 19 us, 4.4 TB/s; 4096x5120 bf16 with GELU and dropout 43 us for 210 MB, 4.9 TB/s,
// in spite of about 1700 cycles a wave for 512 elements).  One row at a time and many waves: with two rows in flight and
// two thirds of the waves the first was 22 us, and the second, then without dz's low part, 40 instead of 34.
// With an activation dz is held halved, before the mask's scale, which wait for the products' epilogue (and the sums'): |act'|
// is at most 1.13, so a finite dy gives a finite dz in its own type.  Its low part is held larger by LO_SCALE: fp16 has no
// numbers below 2^-24, where the low parts of everything below 2^-13 lie; the first part of at most 2^15.2 leaves at most
// 32, 2^15 then.  bf16 has the exponents of fp32.
constexpr float DZ_HELD = 0.5f;
template <typename T> constexpr float LO_SCALE = 1.f;
template <> constexpr float LO_SCALE<half_t> = 1024.f;

// v = hi + lo / LO_SCALE.  Both parts have v's sign and neither is 0 unless v is (or is below the type's smallest number): an
// infinite x or W then gives the infinity of v's sign in both products, where a low part of 0 or of the other sign would
// make it a NaN.  hi is the next number of the type towards 0, so lo is at most one of its steps and rounds to a 2^-15th
// (bf16; fp16 a 2^-21st) of v.  An infinite or NaN v is both.
template <typename T> __device__ __forceinline__ void split_in_two(float v, float& hi, float& lo) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  hi = lo = v;
  if ((u & 0x7FFFFFFFu) - 1u < 0x7F7FFFFFu) {             // finite, not 0
    const float below = __builtin_bit_cast(float, u - 1u);
    if constexpr (__is_same(T, half_t)) hi = (float)__builtin_amdgcn_cvt_pkrtz(below, below)[0];
    else hi = __builtin_bit_cast(float, (u - 1u) & 0xFFFF0000u);
    lo = (v - hi) * LO_SCALE<T>;
  }
}

struct DzParams {
  const void* dy; int64_t lddy;
  const float* preact;          // [M][N], null without an activation
  void* dz;                     // [M][N], null: only the sums are wanted
  void* dz_lo;                  // [M][N] or null: what dz's rounding lost
  float* db_partial;            // [strips][N] or null
  int64_t M, rows_per_strip;
  int N, act, groups;
  float held, db_scale;         // held: what dy is multiplied by
  DropArgs drop;                // (its scale unused)
};

// A block takes `groups` column groups of eight (256 at most) x as many row lanes as its threads give, of one strip:
// consecutive threads read consecutive columns.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(DzParams p) {
  __shared__ float red[256 * 8];
  const int lanes = 256 / p.groups, rl = (int)threadIdx.x / p.groups, cg = (int)threadIdx.x - rl * p.groups;
  const int cgg = (int)blockIdx.x * p.groups + cg, n = cgg * 8;
  const int cnt = p.N - n;
  const int64_t rb = (int64_t)blockIdx.y * p.rows_per_strip;
  const int64_t re = rb + p.rows_per_strip < p.M ? rb + p.rows_per_strip : p.M;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.f;
  unsigned k0 = 0, k1 = 0;
  if (p.drop.thr) drop_key(p.drop, k0, k1);
  if (cnt > 0 && rl < lanes) {
    for (int64_t m = rb + rl; m < re; m += lanes) {
      float v[8], z[8];
      load8<T>((const T*)p.dy + m * p.lddy + n, cnt, v);
      if (p.act != ACT_NONE) load8<float>(p.preact + m * p.N + n, cnt, z);
      if (p.drop.thr) drop8(v, philox8(k0, k1, (unsigned)cgg, (uint64_t)m, p.drop.offset), p.drop.thr, p.held);
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= p.held;
      }
      act_grad_n<T>(z, v, p.act);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += v[e];
      if (p.dz_lo) {
        float lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_in_two<T>(v[e], v[e], lo[e]);
        store8<T>((T*)p.dz_lo + m * p.N + n, cnt, lo);
      }
      if (p.dz) store8<T>((T*)p.dz + m * p.N + n, cnt, v);
    }
  }
  if (!p.db_partial) return;
  if (rl < lanes) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[threadIdx.x * 8 + e] = s[e];
  }
  __syncthreads();
  const int width = p.groups * 8, col0 = (int)blockIdx.x * width;
  for (int c = threadIdx.x; c < width; c += 256) {
    if (col0 + c >= p.N) break;
    float t = 0.f;
    for (int r = 0; r < lanes; ++r) t += red[r * width + c];
    p.db_partial[(size_t)blockIdx.y * p.N + col0 + c] = t * p.db_scale;
  }
}

// ---- host ------------------------------------------------------------------------------------------
// Tile and split of a product: the least of an estimate in microseconds.  A CU works through ceil(workgroups / 256) of
// them, `together` at a time and then the rest, each costing `step` per K-tile of 128 bytes (`alone`, if it is the only
// one, and in between for a few) and its stores (a CU's share of HBM, 20 KB a microsecond); a split contraction stores
// fp32 and pays a join.  Steps measured on MI355X in fp16 with long contractions: 256x320 1.85 (2.8
// with a column operand, not for two: their addresses do not fit the registers beside 160 accumulators), 256x256 1.55
// (1.72 with column operands), 128x128 0.55 with two on a CU, 64x64 0.27 with four; a workgroup that has a CU for itself
// waits for its loads: 0.8 to 1.1 and 0.45 to 0.62, rows before columns, and twice that where the sizes keep the operands
// from LDS-DMA.  twice: the contraction is done a second time, with the low parts of Q.  What the choice is
// worth (us): 8192x4096x4096 217 at 256x256, 284 at 128x128, 546 at 64x64; 4096x5120x1280 54 at 256x320 (256 tiles, one
// round), 72 at 256x256 (two rounds); 320x320x65536 34 at 64x64 in 32 splits, 45 at 256x256 in 64; 308x768x768 6.6 at
// 64x64, 11 at 128x128 in 4 splits, and its dx with the low parts 9 in 4 splits, 16 in one.  fp32 runs at a sixteenth of
// the matrix rate: 128x128 2.3, 64x64 0.65 (alone 0.72).
struct Plan { int bm, bn; unsigned tiles_m, tiles_n, splits; int64_t k_per_split; };

enum Form { FORWARD, GRAD_X, GRAD_W };
// sizes that are no whole 16-byte chunks stay off the large tiles
Plan plan_product(int64_t M, int N, int64_t K, int esize, Form form, bool twice) {
  const bool forward = form == FORWARD;
  const int kt = 128 / esize;
  const int64_t nkt = (K + kt - 1) / kt;
  const bool vec = N % 8 == 0 && (form == GRAD_W ? M : K) * esize % 16 == 0, whole = vec && esize == 2;
  struct Opt { int bm, bn, together; double step, alone; };      // workgroups a CU takes together
  const double step64[3] = {0.40, 0.47, 0.54}, step128[3] = {1.1, 1.25, 1.5};      // not staged by DMA
  const double alone64[2][3] = {{0.8, 1.1, 1.25}, {0.45, 0.58, 0.62}}, alone128[2][3] = {{1.9, 2.4, 3.0}, {0.8, 0.95, 1.1}};
  const Opt opts[4] = {{64, 64, 4, esize == 2 ? (vec ? 0.27 : step64[form]) : 0.65, esize == 2 ? alone64[vec][form] : vec ? 0.72 : 1.3},
                       {128, 128, 2, esize == 2 ? (vec ? 0.55 : step128[form]) : 2.3, esize == 2 ? alone128[vec][form] : vec ? 2.2 : 3.3},
                       {256, 256, 1, forward ? 1.55 : 1.72, 0.0},
                       {256, 320, 1, forward ? 1.85 : 2.8, 0.0}};
  Plan best = {};
  double best_us = 1e30;
  const double out = (double)M * N;
  for (int o = 0; o < (!whole ? 2 : form == GRAD_W ? 3 : 4); ++o) {
    const Opt& t = opts[o];
    const int64_t tm = (M + t.bm - 1) / t.bm, tn = (N + t.bn - 1) / t.bn, tiles = tm * tn;
    if (tiles >= (1ll << 31)) continue;
    for (int64_t s = 1; s <= 64 && s * 2 <= (nkt > 2 ? nkt : 2); s += s < 4 ? 1 : s < 16 ? 2 : 8) {
      if (s > 1 && tiles * s > 1536) break;
      const int64_t per = nkt > 0 ? (nkt + s - 1) / s : 1, used = nkt > 0 ? (nkt + per - 1) / per : 1;
      const int64_t load = (tiles * used + 255) / 256, rest = load % t.together;
      double us = (load - rest) * t.step;
      if (rest) us += t.alone + (rest - 1) * (t.together * t.step - t.alone) / (t.together > 1 ? t.together - 1 : 1);
      us = us * (twice ? 2 * per : per) + load * t.bm * t.bn * (used > 1 ? 4 : esize) / 20e3;
      if (used > 1) us += out * (4.0 * used + esize) / 5.2e6 + 6.0;
      if (us < best_us) {
        best_us = us;
        best = Plan{t.bm, t.bn, (unsigned)tm, (unsigned)tn, (unsigned)used, per * kt};
      }
    }
  }
  return best;
}
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
size_t partial_bytes(const Plan& pl, int64_t M, int N) { return pl.splits > 1 ? up256((size_t)pl.splits * M * N * 4) : 0; }

// rows are whole 16-byte chunks at 16-byte addresses, and the at most 320 of them that a tile takes span less than 2 GiB
bool chunked(const void* p, int64_t ld, int64_t len, int esize) {
  return ((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0 && (len * esize) % 16 == 0 && ld * esize < (1 << 22);
}

template <typename T, bool QC, bool PC, bool VEC>
void launch_tiles(const GemmParams& g, const Plan& pl, hipStream_t stream) {
  const dim3 grid(g.tiles * g.splits + (g.fold.db ? (unsigned)(g.fold.n + DB_COLS - 1) / DB_COLS : 0));
  if constexpr (VEC && sizeof(T) == 2) {
    if (pl.bm == 256) {
      if constexpr (!QC) {
        if (pl.bn == 320) {
          hipLaunchKernelGGL((linear_gemm_kernel<T, 4, 2, 4, 10, QC, PC, true, 2>), grid, dim3(512), 0, stream, g);
          return;
        }
      }
      hipLaunchKernelGGL((linear_gemm_kernel<T, 4, 2, 4, 8, QC, PC, true, 1>), grid, dim3(512), 0, stream, g);
      return;
    }
  }
  if (pl.bm == 128) hipLaunchKernelGGL((linear_gemm_kernel<T, 2, 2, 4, 4, QC, PC, VEC, 0>), grid, dim3(256), 0, stream, g);
  else hipLaunchKernelGGL((linear_gemm_kernel<T, 2, 2, 2, 2, QC, PC, VEC, 0>), grid, dim3(256), 0, stream, g);
}

template <typename T>
int launch_join(const float* partial, unsigned splits, const Epilogue& e, hipStream_t stream) {
  JoinParams j;
  j.partial = partial; j.splits = splits; j.e = e;
  const unsigned groups = (unsigned)(e.N + 7) / 8;
  j.groups = fast_div(groups);
  const int64_t cap = 0x08000000u / groups;
  j.rows_per_y = (unsigned)(e.M < cap ? e.M : cap);
  const unsigned ny = (unsigned)((e.M + j.rows_per_y - 1) / j.rows_per_y);
  // eight threads a group where there are that many splits to read and too few groups to fill the chip with one each
  const int lanes = splits >= 8 && e.M * (int64_t)groups < (1 << 18) ? 8 : 1;
  const dim3 grid((unsigned)(((uint64_t)j.rows_per_y * groups * lanes + 255) / 256), ny);
  if (lanes == 8) hipLaunchKernelGGL((linear_join_kernel<T, 8>), grid, dim3(256), 0, stream, j);
  else hipLaunchKernelGGL((linear_join_kernel<T, 1>), grid, dim3(256), 0, stream, j);
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

// out[m][n] = epilogue(sum_k Q(m, k) P(n, k)), or with a Q2 sum_k (Q / LO_SCALE + Q2)(m, k) P(n, k)
constexpr uint64_t MAX_BLOCKS = (1ull << 32) / 512;      // a launch has less than 2^32 threads: 512 a block, or 256 for two products
struct Product { GemmParams g; Plan pl; bool vec; };
template <typename T, bool QC, bool PC>
int plan_launch(Product* pr, Plan pl, const void* q, const void* q2, int64_t ldq, const void* p, int64_t ldp, int64_t K,
                const Epilogue& e, float* partial, const DbFold& fold) {
  const int sz = (int)sizeof(T);
  pr->vec = chunked(q, ldq, QC ? e.M : K, sz) && ((uintptr_t)q2 & 15) == 0 && chunked(p, ldp, PC ? e.N : K, sz) && e.N % 8 == 0;
  if (!pr->vec && pl.bm == 256) {  // pointers or strides that the sizes do not tell; the splits (and the workspace) stay
    pl.bm = pl.bn = 128;
    pl.tiles_m = (unsigned)((e.M + 127) / 128); pl.tiles_n = (unsigned)((e.N + 127) / 128);
  }
  GemmParams& g = pr->g;
  g.q = (const char*)q; g.q2 = (const char*)q2; g.q_scale = 1.f / LO_SCALE<T>; g.p = (const char*)p; g.fold = fold; g.ldq = ldq; g.ldp = ldp; g.K = K;
  g.k_per_split = pl.k_per_split; g.tiles_n = pl.tiles_n; g.splits = pl.splits; g.e = e;
  const uint64_t total = (uint64_t)pl.tiles_m * pl.tiles_n * pl.splits;
  const uint64_t folds = fold.db ? (uint64_t)(fold.n + DB_COLS - 1) / DB_COLS : 0;
  SDMI_REQUIRE(pl.bm && total + folds < MAX_BLOCKS, "linear_act: %lld x %d outputs are too many", (long long)e.M, e.N);
  g.tiles = pl.tiles_m * pl.tiles_n;
  g.partial = pl.splits > 1 ? partial : nullptr;
  pr->pl = pl;
  return SDMI_OK;
}
template <typename T> int join_splits(const Product& pr, hipStream_t stream) {
  if (pr.g.partial) SDMI_TRY(launch_join<T>(pr.g.partial, pr.g.splits, pr.g.e, stream));
  return SDMI_OK;
}
// sizes, tile and splits, for the profiler's records
void product_label(char (&label)[96], const Product& pr, unsigned more_splits = 0) {
  if (!prof_on()) return;
  const int n = snprintf(label, sizeof(label), "linear M%lld N%d K%lld %dx%d%s/%u", (long long)pr.g.e.M, pr.g.e.N, (long long)pr.g.K,
                         pr.pl.bm, pr.pl.bn, pr.vec ? "" : "u", pr.g.splits);
  if (more_splits) snprintf(label + n, sizeof(label) - n, "+%u", more_splits);      // dx beside dW
}
template <typename T, bool QC, bool PC> int run_product(const Product& pr, hipStream_t stream) {
  char label[96] = "";
  product_label(label, pr);
  {
    ProfScope prof(PROF_OTHER, stream, 2.0 * pr.g.e.M * (double)pr.g.e.N * pr.g.K, 0.0, label);
    if (pr.vec) launch_tiles<T, QC, PC, true>(pr.g, pr.pl, stream);
    else launch_tiles<T, QC, PC, false>(pr.g, pr.pl, stream);
    SDMI_CHECK_HIP(hipGetLastError());
  }
  return join_splits<T>(pr, stream);
}
// dW and dx in one launch, where both take the same one of the small tiles
bool grads_together(const Product& w, const Product& x) {
  return w.pl.bm == x.pl.bm && w.pl.bm <= 128 && w.vec == x.vec;
}
template <typename T, bool VEC> void launch_grads(const Product& w, const Product& x, hipStream_t stream) {
  const dim3 grid(w.g.tiles * w.g.splits + x.g.tiles * x.g.splits + (x.g.fold.db ? (unsigned)(x.g.fold.n + DB_COLS - 1) / DB_COLS : 0));
  if (w.pl.bm == 128) hipLaunchKernelGGL((linear_grads_kernel<T, 4, 4, VEC>), grid, dim3(256), 0, stream, w.g, x.g);
  else hipLaunchKernelGGL((linear_grads_kernel<T, 2, 2, VEC>), grid, dim3(256), 0, stream, w.g, x.g);
}
template <typename T> int run_grads(const Product& w, const Product& x, hipStream_t stream) {
  char label[96] = "";
  product_label(label, w, x.g.splits);
  {
    ProfScope prof(PROF_OTHER, stream, 4.0 * w.g.e.M * (double)w.g.e.N * w.g.K, 0.0, label);
    if (w.vec) launch_grads<T, true>(w, x, stream);
    else launch_grads<T, false>(w, x, stream);
    SDMI_CHECK_HIP(hipGetLastError());
  }
  SDMI_TRY(join_splits<T>(w, stream));
  return join_splits<T>(x, stream);
}

struct BwdLayout { Plan plan_x, plan_w; size_t dz, dz_lo, dbp, px, pw, total; int strips, col_blocks, groups; int64_t rows_per_strip; bool need_dz, split; };
BwdLayout bwd_layout(int64_t M, int K, int N, int act, bool drop, int want, int esize) {
  BwdLayout w;
  size_t o = 0;
  w.need_dz = (act != ACT_NONE || drop) && (want & 3);
  // With an activation dz = dy act'(z) does not fit the tensors' type, and rounded to it adds an error to dx and dw as
  // large as the rounding of their own (error against 64 bits 1.41 times that of an unrounded dz, more where a few
  // entries dominate; 43 % of the entries of 4096x1280x5120 bf16 then are not the ones that 64 bits round to, 0.5 % so).
  // The products therefore take dz in two parts of the type, at any size: how exact a sample's gradient is may not depend
  // on how many others come with it.  The second part costs the products' time again (4096x1280x5120 bf16: 367 us a training pass, 266 with dz rounded).
  w.split = w.need_dz && act != ACT_NONE && esize == 2;
  w.plan_x = plan_product(M, K, N, esize, GRAD_X, w.split);
  w.plan_w = plan_product(N, K, M, esize, GRAD_W, w.split);
  const Plan &px = w.plan_x, &pw = w.plan_w;
  w.dz = o; o += w.need_dz ? up256((size_t)M * N * esize) : 0;
  w.dz_lo = o; o += w.split ? up256((size_t)M * N * esize) : 0;
  // column groups a block takes (all, or an even share), and strips of rows: about 1536 blocks, every row lane at least
  // four rows where there are that many, or fewer if that leaves most of the CUs without a block (308x768 with SiLU 6.9 us
  // in 64 strips, 5.3 in 154)
  const int ncg = (N + 7) / 8;
  w.col_blocks = (ncg + 255) / 256;
  w.groups = (ncg + w.col_blocks - 1) / w.col_blocks;
  const int lanes = 256 / w.groups;
  int64_t strips = 1536 / w.col_blocks;
  if (strips < 1) strips = 1;
  const int64_t by_work = (M + 4 * lanes - 1) / (4 * lanes), by_lane = (M + lanes - 1) / lanes;
  if (strips > by_work) strips = by_work < 256 ? (by_lane < 256 ? by_lane : 256) : by_work;
  if (strips < 1) strips = 1;
  w.rows_per_strip = (M + strips - 1) / strips;
  w.strips = w.rows_per_strip ? (int)((M + w.rows_per_strip - 1) / w.rows_per_strip) : 0;
  w.dbp = o; o += (want & 4) ? up256((size_t)w.strips * N * 4) : 0;
  w.px = o; o += (want & 1) ? partial_bytes(px, M, K) : 0;
  w.pw = o; o += (want & 2) ? partial_bytes(pw, N, K) : 0;
  w.total = o;
  return w;
}

Epilogue plain_out(void* out, int64_t M, int N, float alpha) {
  Epilogue e = {};
  e.out = out; e.ldo = N; e.M = M; e.N = N; e.alpha = alpha;
  return e;
}

template <typename T>
int linear_bwd(const LinearActArgs& a, const BwdLayout& w, const DropArgs& drop, hipStream_t s) {
  char* ws = (char*)a.workspace;
  const void* dz = a.dy;
  int64_t lddz = a.lddy;
  // the mask's scale waits for the products' epilogue: without an activation dz is dy, masked, and nothing is rounded here
  const float held = a.act != ACT_NONE ? DZ_HELD : 1.f, alpha = (drop.thr ? drop.scale : 1.f) / held;
  DbFold fold;
  if (a.rows > 0 && (w.need_dz || a.db)) {
    DzParams d;
    d.dy = a.dy; d.lddy = a.lddy; d.preact = a.act != ACT_NONE ? a.preact : nullptr;
    d.dz = w.need_dz ? ws + w.dz : nullptr;
    d.dz_lo = w.split ? ws + w.dz_lo : nullptr;
    d.db_partial = a.db ? (float*)(ws + w.dbp) : nullptr;
    d.M = a.rows; d.rows_per_strip = w.rows_per_strip; d.N = a.n; d.act = a.act; d.drop = drop; d.groups = w.groups;
    d.held = held; d.db_scale = alpha;
    char label[64] = "";
    if (prof_on()) snprintf(label, sizeof(label), "linear dz %lldx%d", (long long)a.rows, a.n);
    ProfScope prof(PROF_OTHER, s, 0.0, 2.0 * a.rows * (double)a.n * sizeof(T), label);
    hipLaunchKernelGGL(linear_dz_kernel<T>, dim3(w.col_blocks, w.strips), dim3(256), 0, s, d);
    SDMI_CHECK_HIP(hipGetLastError());
    if (w.need_dz) { dz = d.dz; lddz = a.n; }
  }
  if (a.db) { fold.partial = (const float*)(ws + w.dbp); fold.strips = a.rows > 0 ? w.strips : 0; fold.n = a.n; fold.db = a.db; }
  // the products' operands: dz, or its low part and then dz
  const void* q = a.rows > 0 && w.split ? ws + w.dz_lo : dz;
  const void* q2 = q != dz ? dz : nullptr;
  const bool want_x = a.dx && a.rows > 0;
  Product w_, x_;
  if (a.dw)
    SDMI_TRY((plan_launch<T, true, true>(&w_, w.plan_w, q, q2, lddz, a.x, a.ldx, a.rows, plain_out(a.dw, a.n, a.k, alpha),
                                         (float*)(ws + w.pw), fold)));
  if (want_x)
    SDMI_TRY((plan_launch<T, false, true>(&x_, w.plan_x, q, q2, lddz, a.w, a.ldw, a.n, plain_out(a.dx, a.rows, a.k, alpha),
                                          (float*)(ws + w.px), fold)));
  if (a.dw && want_x && grads_together(w_, x_)) {
    w_.g.fold = DbFold();
    SDMI_TRY(run_grads<T>(w_, x_, s));
  } else {
    if (a.dw && want_x) x_.g.fold = DbFold();      // dW's tiles are the smaller ones, which leave a CU room for the fold
    if (a.dw) SDMI_TRY((run_product<T, true, true>(w_, s)));
    if (want_x) SDMI_TRY((run_product<T, false, true>(x_, s)));
  }
  if (a.dw || want_x) fold = DbFold();
  if (fold.db) {
    hipLaunchKernelGGL(linear_db_kernel, dim3((fold.n + DB_COLS - 1) / DB_COLS), dim3(256), 0, s, fold);
    SDMI_CHECK_HIP(hipGetLastError());
  }
  return SDMI_OK;
}

template <typename T>
int linear_few(const LinearActArgs& a, const Epilogue& e, hipStream_t s) {
  GemmParams g = {};
  g.q = (const char*)a.x; g.p = (const char*)a.w; g.ldq = a.ldx; g.ldp = a.ldw; g.K = a.k; g.e = e;
  char label[96] = "";
  if (prof_on()) snprintf(label, sizeof(label), "linear M%lld N%d K%d few", (long long)a.rows, a.n, a.k);
  ProfScope prof(PROF_OTHER, s, 2.0 * a.rows * (double)a.n * a.k, (double)a.n * a.k * sizeof(T), label);
  const dim3 grid((unsigned)(a.n + 15) / 16);
  if (a.rows <= 16) hipLaunchKernelGGL((linear_few_kernel<T, 1>), grid, dim3(512), 0, s, g);
  else hipLaunchKernelGGL((linear_few_kernel<T, 2>), grid, dim3(512), 0, s, g);
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

int check_common(const LinearActArgs& a, const char* who) {
  SDMI_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "%s: bad dtype %d", who, a.dtype);
  SDMI_REQUIRE(a.rows >= 0 && a.k > 0 && a.n > 0, "%s: bad size (%lld rows, %d inputs, %d outputs)", who,
               (long long)a.rows, a.k, a.n);
  SDMI_REQUIRE(a.k <= (1 << 30) && a.n <= (1 << 30), "%s: %d inputs, %d outputs are too many", who, a.k, a.n);
  SDMI_REQUIRE(a.act >= 0 && a.act < ACT_COUNT, "%s: unknown activation %d", who, a.act);
  SDMI_REQUIRE(a.ldx >= 0 && a.ldw >= 0 && a.ldr >= 0 && a.lddy >= 0, "%s: negative row stride", who);
  return SDMI_OK;
}

}  // namespace

int64_t linear_act_workspace_bytes(int64_t rows, int k, int n, int dtype) {
  if (rows <= 0 || k <= 0 || n <= 0 || few_rows(rows, k, n, (int)sdmi_dtype_size(dtype))) return 0;
  return (int64_t)partial_bytes(plan_product(rows, n, k, (int)sdmi_dtype_size(dtype), FORWARD, false), rows, n);
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
  const int esize = (int)sdmi_dtype_size(a.dtype);
  e.bias = a.bias; e.resid = a.resid; e.ldr = a.ldr; e.out = a.out; e.ldo = a.n;
  e.alpha = 1.f; e.preact = a.act != ACT_NONE ? a.preact : nullptr; e.act = a.act; e.M = a.rows; e.N = a.n;
  if (few_rows(a.rows, a.k, a.n, esize)) { SDMI_DISPATCH_DTYPE(a.dtype, T, return linear_few<T>(a, e, stream)); }
  const Plan pl = plan_product(a.rows, a.n, a.k, esize, FORWARD, false);
  const size_t need = partial_bytes(pl, a.rows, a.n);
  SDMI_REQUIRE(need == 0 || a.workspace, "linear_act: this size needs a workspace of %zu bytes", need);
  Product pr;
  SDMI_DISPATCH_DTYPE(a.dtype, T, {
    SDMI_TRY((plan_launch<T, false, false>(&pr, pl, a.x, nullptr, a.ldx, a.w, a.ldw, a.k, e, (float*)a.workspace, DbFold())));
    return run_product<T, false, false>(pr, stream);
  });
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
  }
  const BwdLayout w = bwd_layout(a.rows, a.k, a.n, a.act, drop.thr != 0, want, (int)sdmi_dtype_size(a.dtype));
  SDMI_REQUIRE(a.rows == 0 || w.total == 0 || a.workspace, "linear_act_backward: this size needs a workspace of %zu bytes",
               w.total);
  SDMI_DISPATCH_DTYPE(a.dtype, T, return linear_bwd<T>(a, w, drop, stream));
  return SDMI_OK;
}
