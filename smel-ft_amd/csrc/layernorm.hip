// Layer norm of bf16, fp16 or fp32 rows, forward and backward, with trained weights:
//   y = xhat w + b,  xhat = (x - m) rstd           dx = rstd (g - mean(g) - xhat mean(g xhat)) (+ ds),  g = dy w
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
// and the norm after a residual add, s = round(h + x). fp32 math, one rounding per output. The variance is the mean of
// the squared distances from the mean (the row is in registers, so a second sum over it costs no bytes): a row whose mean
// is large against its spread loses the mean's own fp32 rounding, not the cancellation of two squares.
//
// Layout: a row is split into chunks of 8 elements and belongs to `lpr` threads (a power of two up to 64, or the whole
// block); thread i of a row takes chunks i, i + lpr, .... Chunks are read and written as 16-byte accesses of element
// alignment, which the hardware takes at any address, so odd row lengths and views at any offset run the same code; only
// a row's last, partial chunk goes element by element.
//
// Backward: blocks walk over the rows with a stride, each thread keeping the weights and the dw and db sums of its columns in
// registers and four rows (16-bit) on their way; the block's row groups are joined through LDS in a tree, the blocks' sums go
// to the workspace and a second kernel adds them in block order. No atomics: every result repeats bit for bit. A chunk per
// thread and a block per row, not a wave per row with four chunks: 209 registers there let two waves on a SIMD and every row
// read the weights twice more (32749 x 2048 bf16: 119 us; a block per row 108, with four rows on their way 91; with nontemporal stores 87).
// HBM-bound: forward 4.7 TB/s, backward 4.6 TB/s at 32749 x 2048 bf16 (a copy reaches 5.55).
#include "../../include/smel_norm.h"
#include "abi_util.h"
#include "common.h"
#include "rows.h"

namespace {

constexpr int MAX_COLS = 16384;

struct LnArgs {
  const void *x, *h, *dy, *ds;   // h: fwd with the residual add; dy, ds: bwd
  const void *w, *b;
  void *s, *y, *dx;
  float* stats;                  // [rows][2]: mean, rstd
  float* part;                   // bwd: [blocks][2][cols], null: no weight gradients
  int64_t rows, stride;
  int cols, lpr;
  float eps;
};

template <int DT, int WT, int CPL, int BS, bool ADD>
__global__ __launch_bounds__(BS) void ln_fwd_kernel(LnArgs p) {
  typedef typename El<DT>::T T;
  __shared__ float red[2][16];
  const int lpr = p.lpr, n = p.cols, nch = (n + 7) >> 3;
  const int64_t row = (int64_t)blockIdx.x * (BS / lpr) + threadIdx.x / lpr;
  const int li = threadIdx.x & (lpr - 1);
  const bool live = row < p.rows;
  const int64_t in = (live ? row : 0) * p.stride, out = (live ? row : 0) * (int64_t)n;
  Raw<DT> X[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int ck = li + lpr * k;
    X[k] = Raw<DT>{};
    if (live && ck < nch) {
      X[k] = load8<DT>((const T*)p.x + in, 8 * ck, n);
      if constexpr (ADD) {
        const Raw<DT> H = load8<DT>((const T*)p.h + in, 8 * ck, n);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = X[k].at(j) + H.at(j);
        X[k].set(v);
        store8<DT>((T*)p.s + out, 8 * ck, n, X[k]);
      }
    }
  }
  float sum[1] = {0.f};
#pragma unroll
  for (int k = 0; k < CPL; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[0] += X[k].at(j);   // zero past the row
  row_sums(sum, lpr, red[0]);
  const float mean = sum[0] / (float)n;
  float sq[1] = {0.f};
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int e0 = 8 * (li + lpr * k);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = X[k].at(j) - mean;
      if (e0 + j < n) sq[0] = fmaf(d, d, sq[0]);
    }
  }
  row_sums(sq, lpr, red[1]);
  const float rstd = 1.f / sqrtf(sq[0] / (float)n + p.eps);
  if (!live) return;
  if (li == 0) {
    p.stats[2 * row] = mean;
    p.stats[2 * row + 1] = rstd;
  }
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int ck = li + lpr * k;
    if (ck >= nch) continue;
    float w[8], b[8], v[8];
    weight8<WT>(p.w, 8 * ck, n, 1.f, w);
    weight8<WT>(p.b, 8 * ck, n, 0.f, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fmaf((X[k].at(j) - mean) * rstd, w[j], b[j]);
    Raw<DT> o;
    o.set(v);
    store8<DT>((T*)p.y + out, 8 * ck, n, o);
  }
}

template <int DT, int WT, int CPL, int BS, bool WG>
__global__ __launch_bounds__(BS) void ln_bwd_kernel(LnArgs p) {
  typedef typename El<DT>::T T;
  __shared__ float red[2][32];
  __shared__ float join[WG && BS == 256 ? BS / 2 * CPL * 16 : 1];   // larger blocks are one row's
  const int lpr = p.lpr, n = p.cols, nch = (n + 7) >> 3;
  const int groups = BS / lpr, grp = threadIdx.x / lpr, li = threadIdx.x & (lpr - 1);
  // the weights stay in registers, but for two chunks of fp32 (1024 threads leave 128 registers: they would spill)
  constexpr bool HOLD = !(CPL == 2 && DT == 2);
  float w[CPL][8], dw[WG ? CPL * 8 : 1], db[WG ? CPL * 8 : 1];
  auto weights = [&](int k) {
    const int ck = li + lpr * k;
    weight8<WT>(ck < nch ? p.w : nullptr, 8 * ck, n, 1.f, w[k]);
  };
  if constexpr (HOLD)
#pragma unroll
    for (int k = 0; k < CPL; ++k) weights(k);
  if constexpr (WG)
#pragma unroll
    for (int i = 0; i < CPL * 8; ++i) dw[i] = db[i] = 0.f;
  // PF rows on their way: buffer f is refilled as soon as its row is done with, PF - 1 rows before it is used again
  constexpr int PF = CPL == 2 ? 1 : DT == 2 ? 2 : 4;
  struct Row {
    Raw<DT> x[CPL], d[CPL];
    float mean, rstd;
  } buf[PF];
  auto fetch = [&](Row& b, int64_t row) {
    const bool ok = row < p.rows;
    const int64_t in = (ok ? row : 0) * p.stride, out = (ok ? row : 0) * (int64_t)n;
    b.mean = ok ? p.stats[2 * row] : 0.f;
    b.rstd = ok ? p.stats[2 * row + 1] : 0.f;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int ck = li + lpr * k;
      b.x[k] = b.d[k] = Raw<DT>{};
      if (ok && ck < nch) {
        b.x[k] = load8<DT>((const T*)p.x + in, 8 * ck, n);
        b.d[k] = load8<DT>((const T*)p.dy + out, 8 * ck, n);
      }
    }
  };
  auto one = [&](Row& b, int64_t row, float* rd) {
    const bool live = row < p.rows;
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      if constexpr (!HOLD) weights(k);
#pragma unroll
      for (int j = 0; j < 8; ++j) {   // d is zero past the row and past the last row
        const float d = b.d[k].at(j), xhat = (b.x[k].at(j) - b.mean) * b.rstd;
        const float g = d * w[k][j];
        sums[0] += g;
        sums[1] = fmaf(g, xhat, sums[1]);
        if constexpr (WG) {
          dw[k * 8 + j] = fmaf(d, xhat, dw[k * 8 + j]);
          db[k * 8 + j] += d;
        }
      }
    }
    row_sums(sums, lpr, rd);
    if (!live || !p.dx) return;
    const int64_t out = row * (int64_t)n;
    const float mg = sums[0] / (float)n, mgx = sums[1] / (float)n;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int ck = li + lpr * k;
      if (ck >= nch) continue;
      if constexpr (!HOLD) weights(k);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xhat = (b.x[k].at(j) - b.mean) * b.rstd;
        v[j] = b.rstd * (b.d[k].at(j) * w[k][j] - mg - xhat * mgx);
      }
      if (p.ds) {
        const Raw<DT> S = load8<DT>((const T*)p.ds + out, 8 * ck, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += S.at(j);
      }
      Raw<DT> o;
      o.set(v);
      store8<DT>((T*)p.dx + out, 8 * ck, n, o);
    }
  };
  const int64_t step = (int64_t)gridDim.x * groups, r1 = (int64_t)blockIdx.x * groups;
#pragma unroll
  for (int f = 0; f < PF; ++f) fetch(buf[f], r1 + f * step + grp);
  // every thread of the block takes the same number of turns (row_sums has a barrier); the sums' buffers alternate: a row's
  // readers are done before the next but one writes
  int par = 0;
  for (int64_t r0 = r1; r0 < p.rows; r0 += PF * step)
#pragma unroll
    for (int f = 0; f < PF; ++f) {
      const int64_t row = r0 + f * step;
      if (row >= p.rows) break;
      one(buf[f], row + grp, red[par]);
      par ^= 1;
      fetch(buf[f], row + PF * step + grp);
    }
  if constexpr (WG) {
    for (int half = groups / 2; half >= 1; half /= 2) {
      __syncthreads();
      float* const slot = join + (int64_t)((grp - half) * lpr + li) * (CPL * 16);
      if (grp >= half && grp < 2 * half)
#pragma unroll
        for (int i = 0; i < CPL * 8; ++i) {
          slot[i] = dw[i];
          slot[CPL * 8 + i] = db[i];
        }
      __syncthreads();
      if (grp < half) {
        const float* const from = join + (int64_t)(grp * lpr + li) * (CPL * 16);
#pragma unroll
        for (int i = 0; i < CPL * 8; ++i) {
          dw[i] += from[i];
          db[i] += from[CPL * 8 + i];
        }
      }
    }
    if (grp == 0) {
      float* const o = p.part + (int64_t)blockIdx.x * 2 * n;
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        const int e = 8 * (li + lpr * k);
        if (e >= n) continue;
        Raw<2> a, b;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          a.q[j >> 2][j & 3] = __float_as_uint(dw[k * 8 + j]);
          b.q[j >> 2][j & 3] = __float_as_uint(db[k * 8 + j]);
        }
        store8<2, true>(o, e, n, a);
        store8<2, true>(o + n, e, n, b);
      }
    }
  }
}

// columns of part [blocks][2 n] summed: a wave's lanes take 64 columns, the 16 waves a 16th of the blocks each
template <int WT>
__global__ __launch_bounds__(1024) void ln_wsum_kernel(const float* __restrict__ part, int blocks, int n, void* dw, void* db) {
  typedef typename El<WT>::T T;
  __shared__ float red[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  float v = 0.f;
  if (c < 2 * n)
#pragma unroll 8
    for (int r = wave; r < blocks; r += 16) v += part[(int64_t)r * 2 * n + c];
  red[wave][threadIdx.x & 63] = v;
  __syncthreads();
  if (wave != 0 || c >= 2 * n) return;
  for (int k = 1; k < 16; ++k) v += red[k][threadIdx.x];
  T* const o = (T*)(c < n ? dw : db);
  if (!o) return;
  const int e = c < n ? c : c - n;
  if constexpr (WT == 2)
    o[e] = v;
  else
    o[e] = (T)enc<WT>(v);
}

// ------------------------------------------------------------------------------------------------ host

struct Shape {
  int lpr, cpl, bs;
};
// Forward. Rows of 513 to 2048 columns: a wave each, whose four chunks a lane hide the latency without a barrier, or, where
// there are under 4096 of them, a block each (23 x 2048: 5.6 -> 4.4 us; 32749 rows: 79 us, a wave each 56)
Shape fwd_shape(int64_t rows, int64_t cols) {
  const int nch = (int)((cols + 7) / 8);   // <= 2048
  Shape s{1, 1, 256};
  while (s.lpr < nch && s.lpr < 64) s.lpr *= 2;
  if (nch > 256 || (nch > 64 && rows < 4096)) s.lpr = 256;
  if (nch > 1024) s.lpr = s.bs = 1024;
  while (s.cpl * s.lpr < nch) s.cpl *= 2;   // <= 4
  return s;
}
// backward: a chunk per thread where 1024 threads reach (the weights, their sums and the next row stay in registers)
Shape bwd_shape(int64_t cols) {
  const int nch = (int)((cols + 7) / 8);
  Shape s{1, 1, 256};
  while (s.lpr < nch && s.lpr < 1024) s.lpr *= 2;
  if (s.lpr > 256) s.bs = s.lpr;
  while (s.cpl * s.lpr < nch) s.cpl *= 2;   // <= 2
  return s;
}
// blocks of the backward: its weight sums cost 16 bytes a column and block
int64_t bwd_blocks(int64_t rows, int64_t cols) {
  const Shape s = bwd_shape(cols);
  const int64_t turns = (rows + s.bs / s.lpr - 1) / (s.bs / s.lpr);
  // three blocks a CU of 256 threads, two of 512, one of 1024, with two rows each at least. 32749 x 2048 bf16: 112 us with 512
  // blocks, 87 with 768, 79 with 1024 (and 0.7 us more for their sums; 4092 x 2048 with the add 18.7 and 4.5 with 768, 18.4 and 5.4); 4092 x 2816 fp32: 36 with 384, 33 with 512, 44 with 640
  const int64_t most = s.bs == 256 ? 768 : s.bs == 512 ? 512 : 256, g = (turns + 1) / 2;
  return g < most ? g : most;
}

template <int DT, int WT, int CPL, int BS>
int launch_fwd(const LnArgs& p, hipStream_t stream) {
  const int64_t rpb = BS / p.lpr, blocks = (p.rows + rpb - 1) / rpb;
  SMEL_REQUIRE(blocks * BS < (int64_t)1 << 32, SMEL_EUNSUPPORTED, "layernorm_fwd: %lld rows is too many", (long long)p.rows);
  if (p.h) ln_fwd_kernel<DT, WT, CPL, BS, true><<<(unsigned)blocks, BS, 0, stream>>>(p);
  else ln_fwd_kernel<DT, WT, CPL, BS, false><<<(unsigned)blocks, BS, 0, stream>>>(p);
  return smel::launch_status();
}
template <int DT, int WT, int CPL, int BS>
int launch_bwd(const LnArgs& p, hipStream_t stream) {
  const unsigned blocks = (unsigned)bwd_blocks(p.rows, p.cols);
  if (p.part) ln_bwd_kernel<DT, WT, CPL, BS, true><<<blocks, BS, 0, stream>>>(p);
  else ln_bwd_kernel<DT, WT, CPL, BS, false><<<blocks, BS, 0, stream>>>(p);
  return smel::launch_status();
}
template <bool FWD, int DT, int WT>
int launch_w(LnArgs& p, hipStream_t st) {
  const Shape s = FWD ? fwd_shape(p.rows, p.cols) : bwd_shape(p.cols);
  p.lpr = s.lpr;
  if constexpr (FWD) {
    if (s.bs == 1024) return launch_fwd<DT, WT, 2, 1024>(p, st);
    return s.cpl == 1 ? launch_fwd<DT, WT, 1, 256>(p, st) : s.cpl == 2 ? launch_fwd<DT, WT, 2, 256>(p, st)
                                                                       : launch_fwd<DT, WT, 4, 256>(p, st);
  } else {
    if (s.bs == 256) return launch_bwd<DT, WT, 1, 256>(p, st);
    if (s.bs == 512) return launch_bwd<DT, WT, 1, 512>(p, st);
    return s.cpl == 1 ? launch_bwd<DT, WT, 1, 1024>(p, st) : launch_bwd<DT, WT, 2, 1024>(p, st);
  }
}
template <bool FWD>
int launch(LnArgs& p, int dtype, int wtype, hipStream_t st) {
  if (dtype == 2) return launch_w<FWD, 2, 2>(p, st);
  if (dtype == 0) return wtype == 2 ? launch_w<FWD, 0, 2>(p, st) : launch_w<FWD, 0, 0>(p, st);
  return wtype == 2 ? launch_w<FWD, 1, 2>(p, st) : launch_w<FWD, 1, 1>(p, st);
}

int check(const char* name, int64_t rows, int64_t cols, int64_t stride, int32_t dtype, int32_t wtype) {
  SMEL_REQUIRE(rows >= 0 && cols >= 1, SMEL_EINVAL, "%s: bad sizes rows=%lld cols=%lld", name, (long long)rows,
               (long long)cols);
  SMEL_REQUIRE(cols <= MAX_COLS, SMEL_EUNSUPPORTED, "%s: %lld columns, at most %d", name, (long long)cols, MAX_COLS);
  SMEL_REQUIRE(rows <= 1 || stride >= cols, SMEL_EINVAL, "%s: row stride %lld < cols %lld", name, (long long)stride,
               (long long)cols);
  SMEL_REQUIRE(dtype >= 0 && dtype <= 2, SMEL_EINVAL, "%s: dtype %d (0 = bf16, 1 = fp16, 2 = fp32)", name, dtype);
  SMEL_REQUIRE(wtype == dtype || wtype == 2, SMEL_EINVAL, "%s: weights of type %d with rows of type %d", name, wtype, dtype);
  return 0;
}

}  // namespace

extern "C" int smel_layernorm_fwd(const void* x, const void* h, int64_t rows, int64_t cols, int64_t x_stride,
                                  const void* w, const void* b, float eps, int32_t dtype, int32_t wtype, void* s, void* y,
                                  float* stats, hipStream_t stream) {
  const int rc = check("layernorm_fwd", rows, cols, x_stride, dtype, wtype);
  if (rc) return rc;
  if (rows == 0) return 0;
  SMEL_REQUIRE(x && y && stats && (!h || s), SMEL_EINVAL, "layernorm_fwd: null pointer");
  LnArgs p{};
  p.x = x;
  p.h = h;
  p.w = w;
  p.b = b;
  p.s = s;
  p.y = y;
  p.stats = stats;
  p.rows = rows;
  p.stride = x_stride;
  p.cols = (int)cols;
  p.eps = eps;
  return launch<true>(p, dtype, wtype, stream);
}

extern "C" int64_t smel_layernorm_bwd_ws_floats(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > MAX_COLS) return 0;
  return bwd_blocks(rows, cols) * 2 * cols;
}

extern "C" int smel_layernorm_bwd(const void* dy, const void* x, int64_t rows, int64_t cols, int64_t x_stride,
                                  const void* w, const float* stats, const void* ds, int32_t dtype, int32_t wtype,
                                  void* dx, void* dw, void* db, float* ws, int64_t ws_floats, hipStream_t stream) {
  const int rc = check("layernorm_bwd", rows, cols, x_stride, dtype, wtype);
  if (rc) return rc;
  const bool wg = dw || db;
  SMEL_REQUIRE(rows == 0 || (dy && x && stats), SMEL_EINVAL, "layernorm_bwd: null pointer");
  const int64_t need = smel_layernorm_bwd_ws_floats(rows, cols);
  SMEL_REQUIRE(!wg || rows == 0 || (ws && ws_floats >= need), SMEL_EINVAL,
               "layernorm_bwd: a workspace of %lld floats is needed (got %lld)", (long long)need, (long long)ws_floats);
  int64_t blocks = 0;
  if (rows > 0 && (wg || dx)) {
    LnArgs p{};
    p.x = x;
    p.dy = dy;
    p.ds = ds;
    p.w = w;
    p.dx = dx;
    p.stats = const_cast<float*>(stats);
    p.part = wg ? ws : nullptr;
    p.rows = rows;
    p.stride = x_stride;
    p.cols = (int)cols;
    const int rl = launch<false>(p, dtype, wtype, stream);
    if (rl) return rl;
    blocks = bwd_blocks(rows, cols);
  }
  if (!wg) return 0;
  const dim3 g((unsigned)((2 * cols + 63) / 64)), b(1024);
  if (wtype == 2) ln_wsum_kernel<2><<<g, b, 0, stream>>>(ws, (int)blocks, (int)cols, dw, db);
  else if (wtype == 0) ln_wsum_kernel<0><<<g, b, 0, stream>>>(ws, (int)blocks, (int)cols, dw, db);
  else ln_wsum_kernel<1><<<g, b, 0, stream>>>(ws, (int)blocks, (int)cols, dw, db);
  return smel::launch_status();
}
