// The norm behind a block, its gate, the residual add and scale, and the norm before the next block, forward and backward:
//   n = x r1 w1',  u = h + g n,  s = round(scale u),  y = s r2 w2'          (r1, r2: 1 / root mean square of x and of s)
//   dS = ds + r2 (q - shat mean(q shat)), q = dy w2';  dh = scale dS;  dn = dh g;  dx = r1 (q1 - xhat mean(q1 xhat)), q1 = dn w1'
//   dw1 = sum dn xhat, dw2 = sum dy shat, dgate = dh n (g'), dscale = sum dS u
// fp32 math, one rounding per output; y is the norm of the rounded s, as the next block reads it.
//
// Both row sums of the backward are taken in one reduction: with e = ds + r2 q, v = g w1' xhat and m2 = mean(q shat),
//   sum(v dS) = sum(v e) - r2 m2 sum(v shat)
// so a row costs one barrier. A gate per token and the scale are factors of the whole row: they stay outside the sums.
//
// Layout: rows.h's chunks of 8, `lpr` threads a row (a power of two, forward up to 64, backward up to 256, or the block). Blocks of the backward walk over
// the rows, the weights and their sums in registers; the blocks' sums are added by a second launch in block order. No atomics: every
// result repeats bit for bit.
// HBM-bound, us at 32749 x 2048 bf16 (a tensor: 134 MB; a copy reaches 5.4 TB/s): forward 95 to 101 (5.3 to 5.6 TB/s), with a gate per
// element 117 (5.7); backward 145 (5.5), with every sum 157, with a gate per element 204 (5.3).
#include "sandwich.h"

namespace {

// A chunk's weights as stored, or ones
template <int WT>
SMEL_DEV Raw<WT> stored8(const void* p, int e0, int n) {
  if (p) return load8<WT>((const typename El<WT>::T*)p, e0, n);
  const float one[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
  Raw<WT> r;
  r.set(one);
  return r;
}

// Weights are loaded with the row where a thread has one or two chunks of it: a lone row waits for one round trip to memory instead of
// three.
template <int DT, int WT, int CPL>
__global__ __launch_bounds__(CPL == 4 ? 512 : 256) void sandwich_fwd_kernel(SwArgs a) {
  typedef typename El<DT>::T T;
  __shared__ float red[2][16];
  const smel_sandwich& p = a.c;
  const int lpr = a.lpr, n = (int)p.cols, nch = (n + 7) >> 3;
  constexpr bool ONE = CPL > 1;       // a row a block, of as many waves as it needs
  const int64_t row = ONE ? blockIdx.x : (int64_t)blockIdx.x * (256 / lpr) + threadIdx.x / lpr;
  const int li = ONE ? threadIdx.x : threadIdx.x & (lpr - 1);
  const bool live = row < p.rows;
  const int64_t r = live ? row : 0, out = r * (int64_t)n;
  constexpr bool EARLY = CPL <= 2;
  const float add1 = p.plus_one && p.w1 ? 1.f : 0.f, add2 = p.plus_one && p.w2 ? 1.f : 0.f;
  Raw<DT> X[CPL], H[CPL], G[CPL];
  Raw<WT> W1[EARLY ? CPL : 1], W2[EARLY ? CPL : 1], GC[EARLY ? CPL : 1];
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int ck = li + lpr * k;
    X[k] = H[k] = G[k] = Raw<DT>{};
    if (EARLY && ck < nch) {
      W1[EARLY ? k : 0] = stored8<WT>(p.w1, 8 * ck, n);
      if (p.pre) W2[EARLY ? k : 0] = stored8<WT>(p.w2, 8 * ck, n);
      if (p.gate_kind == G_CHANNEL) GC[EARLY ? k : 0] = stored8<WT>(p.gate, 8 * ck, n);
    }
    if (live && ck < nch) {
      X[k] = load8<DT>((const T*)p.x + r * p.x_stride, 8 * ck, n);
      H[k] = load8<DT>((const T*)p.h + r * p.h_stride, 8 * ck, n);
      if (p.gate_kind == G_FULL) G[k] = load8<DT>((const T*)p.gate + out, 8 * ck, n);
    }
  }
  const float scale = p.scale ? one_at<DT>(p.scale, 0, p.scale_type == 2) : p.scale_value;
  const float tg = p.gate_kind == G_TOKEN ? gate_of(one_at<DT>(p.gate, r, p.gate_type == 2), p.gate_act) : 1.f;
  float ss[1] = {0.f};
#pragma unroll
  for (int k = 0; k < CPL; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss[0] = fmaf(X[k].at(j), X[k].at(j), ss[0]);   // zero past the row
  row_sums<1, ONE>(ss, lpr, red[0]);
  const float r1 = 1.f / sqrtf(ss[0] / (float)n + p.eps);
  ss[0] = 0.f;
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int ck = li + lpr * k;
    if (!live || ck >= nch) continue;
    float g[8], v[8];
    const Raw<WT> w = EARLY ? W1[EARLY ? k : 0] : stored8<WT>(p.w1, 8 * ck, n);
    if (p.gate_kind == G_CHANNEL) {
      const Raw<WT> c = EARLY ? GC[EARLY ? k : 0] : stored8<WT>(p.gate, 8 * ck, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = gate_of(c.at(j), p.gate_act);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = p.gate_kind == G_FULL ? gate_of(G[k].at(j), p.gate_act) : tg;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = scale * fmaf(g[j], X[k].at(j) * r1 * (w.at(j) + add1), H[k].at(j));
    H[k].set(v);
    store8<DT>((T*)p.s + out, 8 * ck, n, H[k]);
    if (p.pre)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (8 * ck + j < n) ss[0] = fmaf(H[k].at(j), H[k].at(j), ss[0]);
  }
  float r2 = 0.f;
  if (p.pre) {
    row_sums<1, ONE>(ss, lpr, red[1]);
    r2 = 1.f / sqrtf(ss[0] / (float)n + p.eps);
  }
  if (!live) return;
  if (p.stats && li == 0) {
    p.stats[2 * row] = r1;
    p.stats[2 * row + 1] = r2;
  }
  if (!p.pre) return;
#pragma unroll
  for (int k = 0; k < CPL; ++k) {
    const int ck = li + lpr * k;
    if (ck >= nch) continue;
    float v[8];
    const Raw<WT> w = EARLY ? W2[EARLY ? k : 0] : stored8<WT>(p.w2, 8 * ck, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = H[k].at(j) * r2 * (w.at(j) + add2);
    Raw<DT> o;
    o.set(v);
    store8<DT>((T*)p.y + out, 8 * ck, n, o);
  }
}

// columns of part [blocks][nsum n] summed: a wave's lanes take 64 columns, the 16 waves a 16th of the blocks each; the last block
// adds the blocks' sums for dscale
template <int DT, int WT>
__global__ __launch_bounds__(1024) void sandwich_wsum_kernel(SwArgs a, int blocks) {
  __shared__ float red[16][64];
  const smel_sandwich& p = a.c;
  const int n = (int)p.cols, cols = a.nsum * n, wave = threadIdx.x >> 6, l = threadIdx.x & 63;
  const int c = blockIdx.x * 64 + l;
  const bool last = p.dscale && blockIdx.x == gridDim.x - 1;
  if (last) {   // a wave's work
    if (wave != 0) return;
    const double* const u = scale_parts(a, blocks);
    double v = 0;
    for (int r = l; r < blocks; r += 64) v += u[r];
    v = wave_sum64(v);
    if (l != 0) return;
    if (DT == 2 || p.scale_type == 2) ((float*)p.dscale)[0] = (float)v;
    else if constexpr (DT != 2) ((uint16_t*)p.dscale)[0] = (uint16_t)enc<DT>((float)v);
    return;
  }
  float v = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int r = wave; r < blocks; r += 16) v += a.part[(int64_t)r * cols + c];
  red[wave][l] = v;
  __syncthreads();
  if (wave != 0 || c >= cols) return;
  for (int k = 1; k < 16; ++k) v += red[k][l];
  const int which = c / n, e = c - which * n;
  void* const o = which == a.at1 ? p.dw1 : which == a.at2 ? p.dw2 : p.dgate;
  if constexpr (WT == 2)
    ((float*)o)[e] = v;
  else
    ((uint16_t*)o)[e] = (uint16_t)enc<WT>(v);
}

// ------------------------------------------------------------------------------------------------ host

// The threads of a row: a power of two up to a wave, several rows a block, or the block; above 2048 columns two chunks a thread, above
// 4096 four, and as many waves as they need. 4096 x 2816 bf16: 20.9 us, with a chunk a thread 23.2; 8192 x 8192 102 and 120
Shape fwd_shape(int64_t cols) {
  const int nch = (int)((cols + 7) / 8);   // <= 2048
  Shape s{1, nch <= 256 ? 1 : nch <= 512 ? 2 : 4, 256};
  if (nch <= 64)
    while (s.lpr < nch) s.lpr *= 2;
  else if (nch <= 256)
    s.lpr = 256;
  else
    s.lpr = s.bs = ((nch + s.cpl - 1) / s.cpl + 63) / 64 * 64;   // <= 512
  return s;
}

template <int DT, int WT, int CPL>
int launch_fwd(const SwArgs& a, const Shape& s, hipStream_t stream) {
  const int64_t rpb = s.bs / s.lpr, blocks = (a.c.rows + rpb - 1) / rpb;
  SMEL_REQUIRE(blocks * s.bs < (int64_t)1 << 32, SMEL_EUNSUPPORTED, "sandwich_fwd: %lld rows is too many", (long long)a.c.rows);
  sandwich_fwd_kernel<DT, WT, CPL><<<(unsigned)blocks, s.bs, 0, stream>>>(a);
  return smel::launch_status();
}
template <int DT, int WT>
struct Launch {
  static int fwd(SwArgs& a, hipStream_t st) {
    const Shape s = fwd_shape(a.c.cols);
    a.lpr = s.lpr;
    return s.cpl == 1 ? launch_fwd<DT, WT, 1>(a, s, st) : s.cpl == 2 ? launch_fwd<DT, WT, 2>(a, s, st) : launch_fwd<DT, WT, 4>(a, s, st);
  }
  static int bwd(SwArgs& a, hipStream_t st) {
    int64_t blocks = 0;
    if (a.c.rows > 0) {
      const int rc = DT == 0 ? smel::sandwich_bwd_bf16(a, st) : DT == 1 ? smel::sandwich_bwd_f16(a, st) : smel::sandwich_bwd_f32(a, st);
      if (rc) return rc;
      blocks = bwd_blocks(a.c.rows, a.c.cols);
    }
    const int64_t wb = (a.nsum * a.c.cols + 63) / 64 + (a.c.dscale ? 1 : 0);
    if (!wb) return 0;
    sandwich_wsum_kernel<DT, WT><<<(unsigned)wb, 1024, 0, st>>>(a, (int)blocks);
    return smel::launch_status();
  }
};
template <typename F>
int by_type(const smel_sandwich& c, F f) {
  if (c.dtype == 2) return f(Launch<2, 2>());
  if (c.dtype == 0) return c.wtype == 2 ? f(Launch<0, 2>()) : f(Launch<0, 0>());
  return c.wtype == 2 ? f(Launch<1, 2>()) : f(Launch<1, 1>());
}

int check(const char* name, const smel_sandwich* c) {
  SMEL_REQUIRE(c, SMEL_EINVAL, "%s: null call", name);
  SMEL_REQUIRE(c->rows >= 0 && c->cols >= 1, SMEL_EINVAL, "%s: bad sizes rows=%lld cols=%lld", name, (long long)c->rows,
               (long long)c->cols);
  SMEL_REQUIRE(c->cols <= MAX_COLS, SMEL_EUNSUPPORTED, "%s: %lld columns, at most %d", name, (long long)c->cols, MAX_COLS);
  SMEL_REQUIRE(c->rows <= 1 || (c->x_stride >= c->cols && (!c->h || c->h_stride >= c->cols)), SMEL_EINVAL,
               "%s: row strides %lld, %lld < cols %lld", name, (long long)c->x_stride, (long long)c->h_stride, (long long)c->cols);
  SMEL_REQUIRE(c->dtype >= 0 && c->dtype <= 2, SMEL_EINVAL, "%s: dtype %d (0 = bf16, 1 = fp16, 2 = fp32)", name, c->dtype);
  SMEL_REQUIRE(c->wtype == c->dtype || c->wtype == 2, SMEL_EINVAL, "%s: weights of type %d with rows of type %d", name, c->wtype,
               c->dtype);
  SMEL_REQUIRE(c->gate_kind >= 0 && c->gate_kind <= 3 && (c->gate_kind == 0 || c->gate || c->rows == 0), SMEL_EINVAL,
               "%s: gate kind %d", name, c->gate_kind);
  SMEL_REQUIRE(c->gate_kind != G_TOKEN || c->gate_type == c->dtype || c->gate_type == 2, SMEL_EINVAL, "%s: gate of type %d", name,
               c->gate_type);
  SMEL_REQUIRE(!c->scale || c->scale_type == c->dtype || c->scale_type == 2, SMEL_EINVAL, "%s: scale of type %d", name, c->scale_type);
  return 0;
}
void places(SwArgs& a) {
  const bool on[3] = {a.c.dw1 != nullptr, a.c.dw2 != nullptr, a.c.dgate && a.c.gate_kind == G_CHANNEL};
  int at[3];
  for (int i = 0; i < 3; ++i) at[i] = on[i] ? a.nsum++ : -1;
  a.at1 = at[0];
  a.at2 = at[1];
  a.atg = at[2];
}

}  // namespace

extern "C" int smel_sandwich_fwd(const smel_sandwich* call, hipStream_t stream) {
  const int rc = check("sandwich_fwd", call);
  if (rc) return rc;
  if (call->rows == 0) return 0;
  SMEL_REQUIRE(call->x && call->h && call->s && (!call->pre || call->y), SMEL_EINVAL, "sandwich_fwd: null pointer");
  SwArgs a{};
  a.c = *call;
  return by_type(a.c, [&](auto l) { return decltype(l)::fwd(a, stream); });
}

extern "C" int64_t smel_sandwich_bwd_ws_floats(const smel_sandwich* call) {
  if (check("sandwich_bwd", call) || call->rows == 0) return 0;
  SwArgs a{};
  a.c = *call;
  places(a);
  const int64_t blocks = bwd_blocks(a.c.rows, a.c.cols);
  return blocks * a.nsum * a.c.cols + (a.c.dscale ? 2 * blocks + 1 : 0);
}

extern "C" int smel_sandwich_bwd(const smel_sandwich* call, float* ws, int64_t ws_floats, hipStream_t stream) {
  const int rc = check("sandwich_bwd", call);
  if (rc) return rc;
  SMEL_REQUIRE(call->rows == 0 || (call->x && call->stats && (!call->dy || call->s) && (!call->dscale || call->h)), SMEL_EINVAL,
               "sandwich_bwd: null pointer");
  const int64_t need = smel_sandwich_bwd_ws_floats(call);
  SMEL_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 8 == 0 && ws_floats >= need), SMEL_EINVAL,
               "sandwich_bwd: an aligned workspace of %lld floats is needed (got %lld)", (long long)need, (long long)ws_floats);
  SwArgs a{};
  a.c = *call;
  a.part = ws;
  places(a);
  return by_type(a.c, [&](auto l) { return decltype(l)::bwd(a, stream); });
}
