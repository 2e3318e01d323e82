// Orthogonalisation of matrix updates (the LoRA factors') by Newton-Schulz products:
//   X0 = G / (|G|_F + eps),   X <- P X  with  P = a I + b A + c A^2,  A = X X^T   (steps times)
// With the short side r as rows, every P is a polynomial of A0 = X0 X0^T, so the P commute and are symmetric: the products
// run on r x r matrices alone,  A <- P A P,  Q <- P Q,  and the result is  Q G  (Q starts as I / (|G|_F + eps)): G is read
// for A0 and for the last product, whatever the number of steps.
//
// A and Q are kept and multiplied in 64 bits (v_mfma_f64_16x16x4_f64). A holds the squares of the singular values: in 32
// bits those under 2^-12 of the largest would drown in A's rounding, and the products blow such a value up by a = 3.4
// each step (its square's error by a^2); in 64 bits the result is that of the formula to fp32's own rounding. The sums
// of A0 run in 64 bits for the same reason; products of fp32 values are exact there.
//
// The accumulator layout of the f64 instruction (register m of lane l: row 4 m + l / 16, column l % 16) is its layout of
// the operand B at step m of a 16-long contraction, and of the operand A of a symmetric matrix: results are the next
// product's operands as they are.
//
// Kernels: gram (a block per slice of columns: the slice's part of A0's upper tiles), iterate (a block per matrix: sums
// the parts in slice order, runs the steps, writes Q's tiles), apply (a block per slice: Q G). Nothing is atomic: results
// repeat bit for bit.
#include "../../include/smel_ortho.h"
#include "abi_util.h"
#include "common.h"

namespace {

typedef double f64x4_t __attribute__((ext_vector_type(4)));
SMEL_DEV f64x4_t mfma64(double a, double b, f64x4_t c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

constexpr int MAX_R = 128;
constexpr int MAX_JOBS = 40;   // of one launch: the jobs travel as kernel arguments (under 4 KiB)
constexpr int WAVES = 8;       // of a gram or apply block

struct Job {
  const void* x;
  void* y;
  int64_t xb, ld;      // batch stride; stride between lines (a line: the side with unit stride)
  int64_t part0;       // first tile-set slot of the job's parts in the workspace
  int32_t batch, r, n;
  int32_t blk0, mat0;  // first block (gram, apply) and first matrix (iterate, Q)
  int32_t slices;      // of a matrix
  int32_t x_tall;      // 1: the short side has the unit stride in x
  int32_t y_tall;      // 1: the short side is y's last
};
struct Jobs {
  int32_t n, slice;    // jobs; columns of a slice (a multiple of 64)
  int64_t pad_;
  Job j[MAX_JOBS];
};
static_assert(sizeof(Jobs) <= 3584, "kernel arguments");

constexpr int ntiles(int nt) { return nt * (nt + 1) / 2; }
// upper tile k -> (t, u), t <= u, row by row
SMEL_DEV void tile_of(int k, int nt, int& t, int& u) {
  t = 0;
  while (k >= nt - t) {
    k -= nt - t;
    ++t;
  }
  u = t + k;
}
SMEL_DEV int tile_at(int t, int u, int nt) { return t * nt - t * (t - 1) / 2 + (u - t); }   // t <= u

template <int DT>
SMEL_DEV float to_f(uint32_t b) {
  if constexpr (DT == 0) return __uint_as_float(b << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
template <int DT>
struct Elem {
  typedef uint16_t T;
};
template <>
struct Elem<1> {
  typedef float T;
};
template <int DT>
SMEL_DEV float ld_elem(const typename Elem<DT>::T* p) {
  if constexpr (DT == 1)
    return *p;
  else
    return to_f<DT>(*p);
}
template <int DT>
SMEL_DEV void st_elem(typename Elem<DT>::T* p, double v) {
  const float f = (float)v;
  if constexpr (DT == 1) *p = f;
  if constexpr (DT == 0) *p = f2bf(f);
  if constexpr (DT == 2) *p = __builtin_bit_cast(uint16_t, (_Float16)f);
}

// the job of block (or matrix) b; uniform
template <bool MAT>
SMEL_DEV int find_job(const Jobs& js, int b) {
  int k = 0;
  while (k + 1 < js.n && b >= (MAT ? js.j[k + 1].mat0 : js.j[k + 1].blk0)) ++k;
  return k;
}

// columns [j0, j0 + slice) of a matrix as fp32 X[i][j] in LDS, rows [r, 16 NT) and columns past n zero
template <int DT>
SMEL_DEV void load_slice(const Job& J, int mat, int j0, int slice, int rp, float* X, int pitch) {
  typedef typename Elem<DT>::T T;
  const T* const x = (const T*)J.x + mat * J.xb;
  const int nc = min(slice, J.n - j0);
  for (int e = threadIdx.x; e < rp * slice; e += blockDim.x) {
    int i, j;
    if (J.x_tall) {
      j = e / rp;
      i = e % rp;
    } else {
      i = e / slice;
      j = e % slice;
    }
    float v = 0.f;
    if (i < J.r && j < nc) v = ld_elem<DT>(x + (J.x_tall ? (j0 + j) * J.ld + i : i * J.ld + j0 + j));
    X[i * pitch + j] = v;
  }
}

// columns of a slice at most: two blocks on a CU
constexpr int max_slice(int nt) { return nt == 1 ? 1024 : nt == 2 ? 512 : nt == 4 ? 256 : 128; }
constexpr int slice_bytes(int nt) { return 16 * nt * (max_slice(nt) + 20) * 4; }

template <int NT, int DT>
__global__ __launch_bounds__(64 * WAVES) void gram_kernel(Jobs js, double* __restrict__ part) {
  constexpr int NTL = ntiles(NT);
  __shared__ __attribute__((aligned(16))) char smem[slice_bytes(NT)];
  static_assert(slice_bytes(NT) >= NTL * 2048, "room for the column groups' sums");
  constexpr int TG = NT == 8 ? 4 : NT == 4 ? 2 : 1, KG = WAVES / TG, TPW = NTL / TG;
  static_assert(TPW * TG == NTL, "tiles per wave");
  float* const X = (float*)smem;
  const int pitch = js.slice + 20;
  const Job& J = js.j[find_job<false>(js, blockIdx.x)];
  const int lb = blockIdx.x - J.blk0, mat = lb / J.slices, sl = lb % J.slices;
  load_slice<DT>(J, mat, sl * js.slice, js.slice, 16 * NT, X, pitch);
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int tg = wave % TG, kg = wave / TG;
  f64x4_t acc[TPW];
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    acc[k] = f64x4_t{0, 0, 0, 0};
    int t, u;
    tile_of(tg * TPW + k, NT, t, u);
    // 16 columns a step, four to a lane: which columns make one instruction's contraction does not matter
    for (int j = 16 * kg; j < js.slice; j += 16 * KG) {
      const f32x4_t a = *(const f32x4_t*)(X + (16 * t + lo) * pitch + j + 4 * hi);
      const f32x4_t b = *(const f32x4_t*)(X + (16 * u + lo) * pitch + j + 4 * hi);
#pragma unroll
      for (int m = 0; m < 4; ++m) acc[k] = mfma64(a[m], b[m], acc[k]);
    }
  }
  // the column groups' sums, in group order
  f64x4_t* const red = (f64x4_t*)smem;   // [TG][TPW][64]
  double* const out = part + (J.part0 + lb) * (int64_t)(NTL * 256);
  for (int g = 1; g < KG; ++g) {
    __syncthreads();
    if (kg == g)
#pragma unroll
      for (int k = 0; k < TPW; ++k) red[(tg * TPW + k) * 64 + lane] = acc[k];
    __syncthreads();
    if (kg == 0)
#pragma unroll
      for (int k = 0; k < TPW; ++k) acc[k] += red[(tg * TPW + k) * 64 + lane];
  }
  if (kg == 0)
#pragma unroll
    for (int k = 0; k < TPW; ++k) *(f64x4_t*)(out + ((tg * TPW + k) * 64 + lane) * 4) = acc[k];
}

struct Steps {
  int32_t steps;
  double a, b, c, eps;
};

constexpr int TP = 17;   // doubles between the rows of a tile in LDS

// waves of an iterate block, one to three upper tiles each
constexpr int it_waves(int nt) { return nt == 8 ? 12 : nt == 4 ? 10 : nt == 2 ? 3 : 1; }

// element (16 u + 4 m + l / 16, 16 t + l % 16) of a symmetric matrix in upper tiles: at + m * step
SMEL_DEV int frag_at(int u, int t, int nt, int lo, int hi, int& step) {
  if (u <= t) {
    step = 4 * TP;
    return tile_at(u, t, nt) * (16 * TP) + hi * TP + lo;
  }
  step = 4;
  return tile_at(t, u, nt) * (16 * TP) + lo * TP + hi;
}

template <int NT>
__global__ __launch_bounds__(64 * it_waves(NT)) void iterate_kernel(Jobs js, Steps st, const double* __restrict__ part,
                                                                   double* __restrict__ Qout) {
  constexpr int NTL = ntiles(NT), W = it_waves(NT), TPW = NTL / W;
  static_assert(TPW * W == NTL, "tiles per wave");
  __shared__ double buf0[NTL * 16 * TP], buf1[NTL * 16 * TP], trs[NT];
  const Job& J = js.j[find_job<true>(js, blockIdx.x)];
  const int mat = blockIdx.x - J.mat0;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  int tt[TPW], uu[TPW];
  f64x4_t A[TPW], Q[TPW], P[TPW];
#pragma unroll
  for (int k = 0; k < TPW; ++k) {
    tile_of(wave * TPW + k, NT, tt[k], uu[k]);
    A[k] = f64x4_t{0, 0, 0, 0};
    const double* p = part + (J.part0 + (int64_t)mat * J.slices) * (NTL * 256) + ((wave * TPW + k) * 64 + lane) * 4;
    for (int s = 0; s < J.slices; ++s) A[k] += *(const f64x4_t*)(p + (int64_t)s * (NTL * 256));
    if (tt[k] == uu[k]) {   // the tile's trace: row 4 m + hi, column lo
      double d = 0;
#pragma unroll
      for (int m = 0; m < 4; ++m) d += 4 * m + hi == lo ? A[k][m] : 0.0;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) d += __shfl_xor(d, o, 64);
      if (lane == 0) trs[tt[k]] = d;
    }
  }
  __syncthreads();
  double tr = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) tr += trs[t];
  const double s = 1.0 / (sqrt(tr) + st.eps);
#pragma unroll
  for (int k = 0; k < TPW; ++k)
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      A[k][m] = A[k][m] * s * s;
      Q[k][m] = tt[k] == uu[k] && 4 * m + hi == lo ? s : 0.0;
    }
  auto put = [&](double* buf, const f64x4_t* M) {
#pragma unroll
    for (int k = 0; k < TPW; ++k)
#pragma unroll
      for (int m = 0; m < 4; ++m) buf[(wave * TPW + k) * (16 * TP) + (4 * m + hi) * TP + lo] = M[k][m];
  };
  auto product = [&](const double* M, const double* N, f64x4_t* out) {
#pragma unroll
    for (int k = 0; k < TPW; ++k) {
      f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        int sa, sb;
        const int a = frag_at(u, tt[k], NT, lo, hi, sa), b = frag_at(u, uu[k], NT, lo, hi, sb);
#pragma unroll
        for (int m = 0; m < 4; ++m) acc = mfma64(M[a + m * sa], N[b + m * sb], acc);
      }
      out[k] = acc;
    }
  };
  for (int it = 0; it < st.steps; ++it) {
    put(buf0, A);
    __syncthreads();
    f64x4_t S[TPW];
    product(buf0, buf0, S);
#pragma unroll
    for (int k = 0; k < TPW; ++k)
#pragma unroll
      for (int m = 0; m < 4; ++m)
        P[k][m] = st.b * A[k][m] + st.c * S[k][m] + (tt[k] == uu[k] && 4 * m + hi == lo ? st.a : 0.0);
    put(buf1, P);
    __syncthreads();
    if (it + 1 < st.steps) {
      product(buf0, buf1, S);   // A P
      __syncthreads();
      put(buf0, S);
      __syncthreads();
      product(buf0, buf1, A);   // A P P
    }
    __syncthreads();
    put(buf0, Q);
    __syncthreads();
    product(buf0, buf1, Q);
    __syncthreads();
  }
  // Q's tiles, both triangles, in the operand layout: tile (u, t) register m of lane l = Q[16 u + 4 m + hi][16 t + lo]
  put(buf0, Q);
  __syncthreads();
  double* const out = Qout + (int64_t)blockIdx.x * (NT * NT * 256);
  for (int k = wave; k < NT * NT; k += W) {
    int sa;
    const int a = frag_at(k / NT, k % NT, NT, lo, hi, sa);
    f64x4_t q;
#pragma unroll
    for (int m = 0; m < 4; ++m) q[m] = buf0[a + m * sa];
    *(f64x4_t*)(out + (k * 64 + lane) * 4) = q;
  }
}

template <int NT, int DT>
__global__ __launch_bounds__(64 * WAVES) void apply_kernel(Jobs js, const double* __restrict__ Qin) {
  __shared__ __attribute__((aligned(16))) char smem[slice_bytes(NT)];
  typedef typename Elem<DT>::T T;
  constexpr int CG = WAVES / NT;   // column groups; a wave owns one tile of rows
  float* const X = (float*)smem;
  const int pitch = js.slice + 20;
  const Job& J = js.j[find_job<false>(js, blockIdx.x)];
  const int lb = blockIdx.x - J.blk0, mat = lb / J.slices, j0 = lb % J.slices * js.slice;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
  const int t = wave % NT, cg = wave / NT;
  f64x4_t q[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u)
    q[u] = *(const f64x4_t*)(Qin + (int64_t)(J.mat0 + mat) * (NT * NT * 256) + ((u * NT + t) * 64 + lane) * 4);
  load_slice<DT>(J, mat, j0, js.slice, 16 * NT, X, pitch);
  __syncthreads();
  const int nc = min(js.slice, J.n - j0);
  T* const y = (T*)J.y + (int64_t)mat * J.r * J.n;
  for (int j = 16 * cg; j < nc; j += 16 * CG) {
    f64x4_t acc = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const double x = X[(16 * u + 4 * m + hi) * pitch + j + lo];
        acc = J.y_tall ? mfma64(x, q[u][m], acc) : mfma64(q[u][m], x, acc);
      }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if (J.y_tall) {   // row: column j + 4 m + hi of the matrix, column: row 16 t + lo
        const int c = j + 4 * m + hi, i = 16 * t + lo;
        if (c < nc && i < J.r) st_elem<DT>(y + (int64_t)(j0 + c) * J.r + i, acc[m]);
      } else {
        const int c = j + lo, i = 16 * t + 4 * m + hi;
        if (c < nc && i < J.r) st_elem<DT>(y + (int64_t)i * J.n + j0 + c, acc[m]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ host

int nt_of(int64_t r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }

int check(const smel_ortho_job* jobs, int32_t n) {
  SMEL_REQUIRE(n >= 0 && (jobs || n == 0), SMEL_EINVAL, "orthogonalize: null jobs");
  for (int k = 0; k < n; ++k) {
    const smel_ortho_job& j = jobs[k];
    SMEL_REQUIRE(j.batch >= 0 && j.rows >= 0 && j.cols >= 0, SMEL_EINVAL, "orthogonalize: job %d has a negative size", k);
    if (j.batch == 0 || j.rows == 0 || j.cols == 0) continue;
    SMEL_REQUIRE(j.rows <= MAX_R || j.cols <= MAX_R, SMEL_EUNSUPPORTED,
                 "orthogonalize: a %lld x %lld matrix, the short side is at most %d", (long long)j.rows, (long long)j.cols, MAX_R);
    SMEL_REQUIRE(j.rows < (int64_t)1 << 30 && j.cols < (int64_t)1 << 30 && j.batch < (int64_t)1 << 30, SMEL_EUNSUPPORTED,
                 "orthogonalize: job %d has a side of 2^30 or more", k);
    SMEL_REQUIRE(j.dtype >= 0 && j.dtype <= 2, SMEL_EINVAL, "orthogonalize: dtype %lld (0 = bf16, 1 = fp32, 2 = fp16)",
                 (long long)j.dtype);
    SMEL_REQUIRE(j.x && j.y, SMEL_EINVAL, "orthogonalize: null pointer");
    const int es = j.dtype == 1 ? 4 : 2;
    SMEL_REQUIRE((uintptr_t)j.x % es == 0 && (uintptr_t)j.y % es == 0, SMEL_EINVAL, "orthogonalize: misaligned pointer");
    SMEL_REQUIRE(j.x_row >= 0 && j.x_col >= 0 && j.x_batch >= 0, SMEL_EINVAL, "orthogonalize: negative stride");
    SMEL_REQUIRE((j.cols == 1 || j.x_col == 1) || (j.rows == 1 || j.x_row == 1), SMEL_EINVAL,
                 "orthogonalize: neither side of job %d has unit stride", k);
  }
  return 0;
}

struct Plan {
  Jobs js;
  int64_t blocks, mats, parts;   // blocks of gram and apply, matrices, tile sets of the parts
};

// the jobs of one (tiles a side, dtype), MAX_JOBS at a time from `from`; returns the index behind the last job taken
int fill(const smel_ortho_job* jobs, int32_t n, int from, int nt, int dt, Plan& p) {
  p.js.n = 0;
  p.blocks = p.mats = p.parts = 0;
  int end = from;
  int64_t cols = 0;
  int taken[MAX_JOBS];
  for (; end < n && p.js.n < MAX_JOBS; ++end) {
    const smel_ortho_job& j = jobs[end];
    if (j.batch == 0 || j.rows == 0 || j.cols == 0 || j.dtype != dt) continue;
    const int64_t r = j.rows < j.cols ? j.rows : j.cols;
    if (nt_of(r) != nt) continue;
    taken[p.js.n++] = end;
    cols += j.batch * (j.rows < j.cols ? j.cols : j.rows);
  }
  int slice = max_slice(nt);
  while (slice > 128 && cols / slice < 512) slice /= 2;
  p.js.slice = slice;
  for (int k = 0; k < p.js.n; ++k) {
    const smel_ortho_job& j = jobs[taken[k]];
    Job& o = p.js.j[k];
    const bool wide = j.rows <= j.cols;   // the short side is the rows
    o.x = j.x;
    o.y = j.y;
    o.xb = j.x_batch;
    o.r = (int32_t)(wide ? j.rows : j.cols);
    o.n = (int32_t)(wide ? j.cols : j.rows);
    o.batch = (int32_t)j.batch;
    o.y_tall = !wide;
    const bool last = j.cols == 1 || j.x_col == 1;   // lines run along the last side
    if (last && !(j.cols == 1 && j.rows > 1 && j.x_row == 1)) {
      o.ld = j.x_row;
      o.x_tall = !wide;
    } else {
      o.ld = j.x_col;
      o.x_tall = wide;
    }
    o.slices = (o.n + slice - 1) / slice;
    o.blk0 = (int32_t)p.blocks;
    o.mat0 = (int32_t)p.mats;
    o.part0 = p.blocks;
    p.blocks += j.batch * o.slices;
    p.mats += j.batch;
    if (p.blocks >= (int64_t)1 << 22) return -1;   // 768 threads each: a launch takes fewer than 2^32
  }
  p.parts = p.blocks;
  return end;
}

int64_t part_bytes(const Plan& p, int nt) { return p.parts * ntiles(nt) * 2048; }
int64_t q_bytes(const Plan& p, int nt) { return p.mats * nt * nt * 2048; }

template <int NT, int DT>
int run(const Plan& p, const Steps& st, void* ws, hipStream_t stream) {
  const Jobs& js = p.js;
  double* const part = (double*)ws;
  double* const Q = (double*)((char*)ws + part_bytes(p, NT));
  gram_kernel<NT, DT><<<(unsigned)p.blocks, 64 * WAVES, 0, stream>>>(js, part);
  iterate_kernel<NT><<<(unsigned)p.mats, 64 * it_waves(NT), 0, stream>>>(js, st, part, Q);
  apply_kernel<NT, DT><<<(unsigned)p.blocks, 64 * WAVES, 0, stream>>>(js, Q);
  return smel::launch_status();
}
template <int NT>
int run_dt(const Plan& p, int dt, const Steps& st, void* ws, hipStream_t stream) {
  return dt == 0 ? run<NT, 0>(p, st, ws, stream) : dt == 1 ? run<NT, 1>(p, st, ws, stream) : run<NT, 2>(p, st, ws, stream);
}

// f(plan, nt, dt) for every launch group, in order; stops at the first non-zero result
template <class F>
int each(const smel_ortho_job* jobs, int32_t n, F f) {
  for (int nt = 1; nt <= 8; nt *= 2)
    for (int dt = 0; dt < 3; ++dt)
      for (int at = 0; at < n;) {
        Plan p;
        at = fill(jobs, n, at, nt, dt, p);
        SMEL_REQUIRE(at >= 0, SMEL_EUNSUPPORTED, "orthogonalize: too many matrices in one call");
        if (p.js.n == 0) continue;
        const int rc = f(p, nt, dt);
        if (rc) return rc;
      }
  return 0;
}

int64_t ws_need(const smel_ortho_job* jobs, int32_t n, int& rc) {
  int64_t need = 0;   // the groups run one after the other on one stream and share the workspace
  rc = each(jobs, n, [&](const Plan& p, int nt, int) {
    const int64_t b = part_bytes(p, nt) + q_bytes(p, nt);
    if (b > need) need = b;
    return 0;
  });
  return need;
}

}  // namespace

extern "C" int64_t smel_orthogonalize_ws(const smel_ortho_job* jobs, int32_t n_jobs) {
  if (check(jobs, n_jobs)) return -1;
  int rc = 0;
  const int64_t need = ws_need(jobs, n_jobs, rc);
  return rc ? -1 : need;
}

extern "C" int smel_orthogonalize(const smel_ortho_job* jobs, int32_t n_jobs, int32_t steps, double a, double b,
                                  double c, double eps, void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check(jobs, n_jobs);
  if (rc) return rc;
  SMEL_REQUIRE(steps >= 0 && steps <= 64, SMEL_EINVAL, "orthogonalize: %d steps (0 to 64)", steps);
  SMEL_REQUIRE(eps >= 0, SMEL_EINVAL, "orthogonalize: eps %g", eps);
  const int64_t need = ws_need(jobs, n_jobs, rc);
  if (rc) return rc;
  SMEL_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need), SMEL_EINVAL,
               "orthogonalize: a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need,
               (long long)ws_bytes);
  const Steps st{steps, a, b, c, eps};
  return each(jobs, n_jobs, [&](const Plan& p, int nt, int dt) {
    return nt == 1 ? run_dt<1>(p, dt, st, ws, stream) : nt == 2 ? run_dt<2>(p, dt, st, ws, stream)
           : nt == 4 ? run_dt<4>(p, dt, st, ws, stream) : run_dt<8>(p, dt, st, ws, stream);
  });
}
