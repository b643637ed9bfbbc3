// Dropout with the counter-based mask of act_drop.h, optionally added to a residual:
//   out[r][c] = [resid[r][c] +] keep(r, c) x[r][c] / (1 - p)
// The backward pass is the same kernel on the gradient.  HBM-bound: a thread owns eight consecutive columns (one
// generator call, one 16-byte load and store of a 16-bit type), and as many threads as that takes: 65536x1280 bf16 58 to
// 62 us, 5.4 to 5.8 TB/s (a copy of 1 GiB runs at 5.2); 9217x333 fp16, every row at another address, 5.6 us (2.2 TB/s);
// 256x64 fp32 2.5 us, a launch.
#include "act_drop.h"
#include "ops.h"
#include <stdio.h>

namespace {

struct DropoutParams {
  const void* x; const void* resid; void* out;
  int64_t ldx, ldr, ldo, rows;
  int cols;
  unsigned rows_per_y;          // rows of one blockIdx.y: rows_per_y * groups stays below 2^31
  FastDiv groups;               // eight-column groups per row
  DropArgs drop;
};

template <typename T, bool RESID>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutParams p) {
  const int64_t row_base = (int64_t)blockIdx.y * p.rows_per_y;
  const int64_t left = p.rows - row_base;
  const unsigned rows = left < (int64_t)p.rows_per_y ? (unsigned)left : p.rows_per_y;
  const unsigned total = rows * p.groups.d;
  unsigned k0, k1;
  drop_key(p.drop, k0, k1);
  for (unsigned i = blockIdx.x * 256u + threadIdx.x; i < total; i += gridDim.x * 256u) {
    const unsigned r = div_by(i, p.groups), j = i - r * p.groups.d;
    const int64_t row = row_base + r;
    const int c = (int)j * 8, n = p.cols - c;
    float v[8];
    load8<T>((const T*)p.x + row * p.ldx + c, n, v);
    float w[8];
    if (RESID) load8<T>((const T*)p.resid + row * p.ldr + c, n, w);
    drop8(v, philox8(k0, k1, j, (uint64_t)row, p.drop.offset), p.drop.thr, p.drop.scale);
    if (RESID) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[e];
    }
    store8<T>((T*)p.out + row * p.ldo + c, n, v);
  }
}

template <typename T>
int launch_dropout(const DropoutArgs& a, const DropArgs& drop, hipStream_t stream) {
  DropoutParams p;
  p.x = a.x; p.resid = a.resid; p.out = a.out; p.ldx = a.ldx; p.ldr = a.ldr; p.ldo = a.cols;
  p.rows = a.rows; p.cols = a.cols; p.drop = drop;
  const unsigned groups = (unsigned)(a.cols + 7) / 8;
  p.groups = fast_div(groups);
  const int64_t cap = (int64_t)(0x70000000u / groups);
  p.rows_per_y = (unsigned)(a.rows < cap ? a.rows : cap);
  const int64_t ny = (a.rows + p.rows_per_y - 1) / p.rows_per_y;
  SDMI_REQUIRE(ny <= 65535, "dropout: %lld rows of %d columns are too many", (long long)a.rows, a.cols);
  const unsigned blocks = (unsigned)(((uint64_t)p.rows_per_y * groups + 255) / 256);
  char label[64] = "";
  if (prof_on()) snprintf(label, sizeof(label), "dropout %lldx%d", (long long)a.rows, a.cols);
  ProfScope prof(PROF_OTHER, stream, 0.0, (a.resid ? 3.0 : 2.0) * a.rows * (double)a.cols * sizeof(T), label);
  const dim3 grid(blocks, (unsigned)ny);
  if (a.resid) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, stream, p);
  SDMI_CHECK_HIP(hipGetLastError());
  return SDMI_OK;
}

}  // namespace

int dropout(const DropoutArgs& a, hipStream_t stream) {
  SDMI_REQUIRE(a.rows >= 0 && a.cols >= 0, "dropout: negative size");
  SDMI_REQUIRE(a.cols <= (1 << 30), "dropout: rows of %d columns are too long", a.cols);
  SDMI_REQUIRE(a.ldx >= 0 && a.ldr >= 0, "dropout: negative row stride");
  DropArgs drop;
  SDMI_TRY(drop_args(&drop, a.p, a.seed, a.seed_dev, a.offset, "dropout"));
  SDMI_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "dropout: bad dtype %d", a.dtype);
  if (a.rows == 0 || a.cols == 0) return SDMI_OK;
  SDMI_REQUIRE(a.x && a.out, "dropout: null pointer");
  SDMI_DISPATCH_DTYPE(a.dtype, T, return launch_dropout<T>(a, drop, stream));
  return SDMI_OK;
}
