// What the kernels of the norms around a residual add share (sandwich.hip, sandwich_bwd_*.hip).
#pragma once
#include "../../include/smel_norm.h"
#include "abi_util.h"
#include "common.h"
#include "rows.h"

struct SwArgs {
  smel_sandwich c;
  float* part;      // [blocks][nsum cols], then (8-byte aligned) a double a block for dscale
  int lpr, nsum, at1, at2, atg;   // sums of a column: their number and places (-1: not wanted)
};

namespace smel {
// The backward's kernel for each type of rows: a file each, so that they are built side by side
int sandwich_bwd_bf16(SwArgs& a, hipStream_t stream);
int sandwich_bwd_f16(SwArgs& a, hipStream_t stream);
int sandwich_bwd_f32(SwArgs& a, hipStream_t stream);
}  // namespace smel

namespace {

constexpr int MAX_COLS = 16384;
enum { G_NONE = 0, G_CHANNEL = 1, G_TOKEN = 2, G_FULL = 3 };

// The sigmoid and its slope s (1 - s) from q = e^-|z|, each exact to a few ulps: e^x as 2^(t + c), t + c = x log2 e in two floats
// (c of an x that is finite: where it differs, 2^t is 0). NaN stays NaN.
SMEL_DEV float exp_neg_abs(float z) {
  const float x = -fabsf(z), y = fmaxf(x, -126.f), t = y * 1.44269502f;
  const float c = fmaf(y, 1.92596300e-8f, fmaf(y, 1.44269502f, -t));
  const float r = __builtin_amdgcn_exp2f(x * 1.44269502f);
  return fmaf(r, c * 0.693147182f, r);
}
SMEL_DEV float gate_of(float z, int act) {
  if (!act) return z;
  const float q = exp_neg_abs(z), a = __builtin_amdgcn_rcpf(1.f + q);
  return z < 0.f ? q * a : a;
}
SMEL_DEV float gate_of(float z, int act, float& slope) {
  slope = 1.f;
  if (!act) return z;
  const float q = exp_neg_abs(z), a = __builtin_amdgcn_rcpf(1.f + q);
  slope = q * a * a;
  return z < 0.f ? q * a : a;
}
SMEL_DEV float gate_slope(float z, int act) {
  float s;
  gate_of(z, act, s);
  return s;
}
// element i of rows' type DT, or of fp32
template <int DT>
SMEL_DEV float one_at(const void* p, int64_t i, bool f32) {
  if (DT == 2 || f32) return ((const float*)p)[i];
  if constexpr (DT != 2) return cvt<DT>(((const uint16_t*)p)[i]);
  return 0.f;
}

SMEL_DEV double* scale_parts(const SwArgs& a, int64_t blocks) {
  return (double*)(a.part + ((blocks * a.nsum * a.c.cols + 1) & ~(int64_t)1));
}
SMEL_DEV double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct Shape {
  int lpr, cpl, bs;
};
// The threads of a row: a power of two up to 256, several rows a block; above 2048 columns the block, as many waves as it needs. A
// chunk per thread, two above 8192 columns. bs: the kernel's most threads.
Shape bwd_shape(int64_t cols) {
  const int nch = (int)((cols + 7) / 8);
  Shape s{1, nch > 1024 ? 2 : 1, 256};
  if (nch <= 256) {
    while (s.lpr < nch) s.lpr *= 2;
    return s;
  }
  s.lpr = ((nch + s.cpl - 1) / s.cpl + 63) / 64 * 64;
  s.bs = s.lpr <= 512 && s.cpl == 1 ? 512 : 1024;
  return s;
}
int64_t bwd_blocks(int64_t rows, int64_t cols) {
  const Shape s = bwd_shape(cols);
  const int64_t rpb = s.bs == 256 ? 256 / s.lpr : 1, turns = (rows + rpb - 1) / rpb;
  const int64_t most = s.bs == 256 ? 768 : s.bs == 512 ? 512 : 256;
  return turns < most ? turns : most;
}

}  // namespace
