// The backward of the norms around a residual add for rows of one type (sandwich.hip has the formulas). HBM-bound.
#pragma once
#include "sandwich.h"

namespace {

// w' of a chunk, or a gate's values; weights of the rows' type or fp32
template <int DT>
SMEL_DEV void chunk_weight8(int wtype, const void* p, int e0, int n, int plus_one, float v[8]) {
  if (wtype == 2) weight8<2>(p, e0, n, 1.f, v);
  else if constexpr (DT != 2) weight8<DT>(p, e0, n, 1.f, v);
  if (plus_one && p)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += 1.f;
}

template <int DT, int CPL, int BS, int GK, bool PRE, bool WG>
__global__ __launch_bounds__(BS, BS == 256 ? 3 : 4) void sandwich_bwd_kernel(SwArgs a) {
  typedef typename El<DT>::T T;
  __shared__ float red[2][48];
  __shared__ float join[WG && BS == 256 ? BS / 2 * CPL * 24 : 1];   // larger blocks are one row's
  __shared__ double joins[16];
  const smel_sandwich& p = a.c;
  const int lpr = a.lpr, n = (int)p.cols, nch = (n + 7) >> 3;
  constexpr bool ONE = BS > 256;      // a row a block, of as many waves as it needs
  const int groups = ONE ? 1 : BS / lpr, grp = ONE ? 0 : threadIdx.x / lpr, li = ONE ? threadIdx.x : threadIdx.x & (lpr - 1);
  const float scale = p.scale ? one_at<DT>(p.scale, 0, p.scale_type == 2) : p.scale_value;
  // The weights stay in registers where a thread has one chunk, and so does the row. 1024 threads leave a thread of two chunks 128
  // registers: the weights are read again after the row's sums, and 16-bit rows too, from the caches (4000 x 16384 bf16 with the
  // weights' sums 363 -> 228 us; fp32 rows are kept: 507 us, read again 599)
  constexpr bool HOLD = CPL == 1, KEEP = HOLD || DT == 2;
  float w1[8], w2[8], gc[8];
  auto weights = [&](int k) {
    const int ck = li + lpr * k;
    chunk_weight8<DT>(p.wtype, ck < nch ? p.w1 : nullptr, 8 * ck, n, p.plus_one, w1);
    if (PRE) chunk_weight8<DT>(p.wtype, ck < nch ? p.w2 : nullptr, 8 * ck, n, p.plus_one, w2);
    if (GK == G_CHANNEL) {
      chunk_weight8<DT>(p.wtype, ck < nch ? p.gate : nullptr, 8 * ck, n, 0, gc);
#pragma unroll
      for (int j = 0; j < 8; ++j) gc[j] = gate_of(gc[j], p.gate_act);
    }
  };
  if constexpr (HOLD) weights(0);
  float sums[WG ? CPL * 24 : 1];   // of a chunk's columns: dw1, dw2, dgate
  double usum = 0;                 // of dS u: its terms cancel, and a block has thousands of them
  if constexpr (WG)
#pragma unroll
    for (int i = 0; i < CPL * 24; ++i) sums[i] = 0.f;
  struct Chunk {
    Raw<DT> x, d, s, y, g;
  };
  auto fetch = [&](Chunk& c, int64_t row, int k) {
    const int ck = li + lpr * k;
    const bool in = row < p.rows && ck < nch;
    const int64_t r = in ? row : 0, out = r * (int64_t)n;
    c.x = c.d = c.s = c.y = c.g = Raw<DT>{};
    if (in) c.x = load8<DT>((const T*)p.x + r * p.x_stride, 8 * ck, n);
    if (in && p.ds) c.d = load8<DT>((const T*)p.ds + out, 8 * ck, n);
    if (PRE && in) {
      c.s = load8<DT>((const T*)p.s + out, 8 * ck, n);
      c.y = load8<DT>((const T*)p.dy + out, 8 * ck, n);
    }
    if (GK == G_FULL && in) c.g = load8<DT>((const T*)p.gate + out, 8 * ck, n);
  };
  auto one = [&](int64_t row, float* rd) {
    const bool live = row < p.rows;
    Chunk chunks[KEEP ? CPL : 1];
    if constexpr (KEEP)
#pragma unroll
      for (int k = 0; k < CPL; ++k) fetch(chunks[k], row, k);
    const float r1 = live ? p.stats[2 * row] : 0.f, r2 = live && PRE ? p.stats[2 * row + 1] : 0.f;
    const bool token = GK == G_TOKEN && p.gate_kind == G_TOKEN;
    const float tz = token && live ? one_at<DT>(p.gate, row, p.gate_type == 2) : 0.f;
    const float tg = token ? gate_of(tz, p.gate_act) : 1.f;
    float gv[GK == G_FULL ? 8 : 1], gs[GK == G_FULL ? 8 : 1];   // a chunk's gate and its slope
    auto gates = [&](const Chunk& c) {
      if constexpr (GK == G_FULL)
#pragma unroll
        for (int j = 0; j < 8; ++j) gv[j] = gate_of(c.g.at(j), p.gate_act, gs[j]);
    };
    auto gate = [&](int j) { return GK == G_CHANNEL ? gc[j] : GK == G_FULL ? gv[j] : 1.f; };
    float abc[PRE ? 3 : 1] = {};
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      Chunk& c = chunks[KEEP ? k : 0];
      if constexpr (!KEEP) fetch(c, row, k);
      if constexpr (!HOLD) weights(k);
      gates(c);
#pragma unroll
      for (int j = 0; j < 8; ++j) {   // x and s are zero past the row and past the last row
        const float v = gate(j) * w1[j] * (c.x.at(j) * r1);
        if constexpr (PRE) {
          const float q = c.y.at(j) * w2[j], sh = c.s.at(j) * r2;
          abc[0] = fmaf(v, fmaf(r2, q, c.d.at(j)), abc[0]);
          abc[1] = fmaf(q, sh, abc[1]);
          abc[2] = fmaf(v, sh, abc[2]);
        } else {
          abc[0] = fmaf(v, c.d.at(j), abc[0]);
        }
      }
    }
    row_sums<PRE ? 3 : 1, ONE>(abc, lpr, rd);
    if constexpr (!KEEP) asm volatile("" ::: "memory");     // the chunks are read again, not kept
    const float m2 = PRE ? r2 * (abc[PRE ? 1 : 0] / (float)n) : 0.f;
    const float vd = scale * (PRE ? abc[0] - m2 * abc[PRE ? 2 : 0] : abc[0]);   // the sum of dh w1' xhat (g)
    const float m1 = tg * vd / (float)n;
    if (!live) return;
    if (token && p.dgate && li == 0) {
      const float d = vd * gate_slope(tz, p.gate_act);
      if (DT == 2 || p.gate_type == 2) ((float*)p.dgate)[row] = d;
      else if constexpr (DT != 2) ((T*)p.dgate)[row] = (T)enc<DT>(d);
    }
    const int64_t out = row * (int64_t)n;
#pragma unroll
    for (int k = 0; k < CPL; ++k) {
      const int ck = li + lpr * k;
      if (ck >= nch) continue;
      Chunk& c = chunks[KEEP ? k : 0];
      if constexpr (!KEEP) fetch(c, row, k);
      if constexpr (!HOLD) {
        weights(k);
        gates(c);
      }
      float dh[8], dx[8], dg[8], u[8], us = 0.f;
      if (p.dscale) {
        const Raw<DT> H = load8<DT>((const T*)p.h + row * p.h_stride, 8 * ck, n);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = H.at(j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g = gate(j), xh = c.x.at(j) * r1;
        float ds = c.d.at(j), sh = 0.f;
        if constexpr (PRE) {
          sh = c.s.at(j) * r2;
          ds = fmaf(r2, c.y.at(j) * w2[j], ds) - m2 * sh;
        }
        dh[j] = scale * ds;
        const float dn = dh[j] * g * tg;
        dx[j] = r1 * (dn * w1[j] - xh * m1);
        dg[j] = dh[j] * xh * w1[j];
        if (p.dscale && 8 * ck + j < n) us = fmaf(ds, fmaf(g * tg, xh * w1[j], u[j]), us);
        if constexpr (WG) {
          sums[k * 24 + j] = fmaf(dn, xh, sums[k * 24 + j]);
          if constexpr (PRE) sums[k * 24 + 8 + j] = fmaf(c.y.at(j), sh, sums[k * 24 + 8 + j]);
          if constexpr (GK == G_CHANNEL) sums[k * 24 + 16 + j] += dg[j];
        }
      }
      usum += (double)us;
      Raw<DT> o;
      if (p.dh) {
        o.set(dh);
        store8<DT>((T*)p.dh + out, 8 * ck, n, o);
      }
      if (p.dx) {
        o.set(dx);
        store8<DT>((T*)p.dx + out, 8 * ck, n, o);
      }
      if (GK == G_FULL && p.dgate) {
#pragma unroll
        for (int j = 0; j < 8; ++j) dg[j] *= gs[j];
        o.set(dg);
        store8<DT>((T*)p.dgate + out, 8 * ck, n, o);
      }
    }
  };
  // every thread of the block takes the same number of turns (row_sums has a barrier); the sums' buffers alternate: a row's
  // readers are done before the next but one writes
  int par = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * groups; r0 < p.rows; r0 += (int64_t)gridDim.x * groups, par ^= 1) {
    one(r0 + grp, red[par]);
  }
  if (p.dscale) {   // the block's sum of dS u
    usum = wave_sum64(usum);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) joins[threadIdx.x >> 6] = usum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < (int)blockDim.x >> 6; ++w) usum += joins[w];
      scale_parts(a, gridDim.x)[blockIdx.x] = usum;
    }
  }
  if constexpr (WG) {
    for (int half = groups / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (grp >= half && grp < 2 * half)
#pragma unroll
        for (int i = 0; i < CPL * 24; ++i) join[((grp - half) * lpr + li) * (CPL * 24) + i] = sums[i];
      __syncthreads();
      if (grp < half)
#pragma unroll
        for (int i = 0; i < CPL * 24; ++i) sums[i] += join[(grp * lpr + li) * (CPL * 24) + i];
    }
    if (grp == 0) {
      float* const o = a.part + (int64_t)blockIdx.x * a.nsum * n;
      const int at[3] = {a.at1, a.at2, a.atg};
#pragma unroll
      for (int k = 0; k < CPL; ++k) {
        const int e = 8 * (li + lpr * k);
        if (e >= n) continue;
        if (GK == G_CHANNEL && p.gate_act) {
          float z[8];
          chunk_weight8<DT>(p.wtype, p.gate, e, n, 0, z);
#pragma unroll
          for (int j = 0; j < 8; ++j) sums[k * 24 + 16 + j] *= gate_slope(z[j], 1);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (at[i] < 0) continue;
          Raw<2> v;
          v.set(sums + k * 24 + 8 * i);
          store8<2, true>(o + (int64_t)at[i] * n, e, n, v);
        }
      }
    }
  }
}

template <int DT, int CPL, int BS, int GK, bool PRE>
int launch_bwd_sums(const SwArgs& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)bwd_blocks(a.c.rows, a.c.cols);
  if (a.nsum) sandwich_bwd_kernel<DT, CPL, BS, GK, PRE, true><<<blocks, BS == 256 ? 256 : a.lpr, 0, stream>>>(a);
  else sandwich_bwd_kernel<DT, CPL, BS, GK, PRE, false><<<blocks, BS == 256 ? 256 : a.lpr, 0, stream>>>(a);
  return smel::launch_status();
}
template <int DT, int CPL, int BS, int GK>
int launch_bwd_gate(const SwArgs& a, hipStream_t stream) {
  return a.c.dy ? launch_bwd_sums<DT, CPL, BS, GK, true>(a, stream) : launch_bwd_sums<DT, CPL, BS, GK, false>(a, stream);
}
template <int DT, int CPL, int BS>
int launch_bwd(const SwArgs& a, hipStream_t stream) {
  switch (a.c.gate_kind) {
    case G_CHANNEL: return launch_bwd_gate<DT, CPL, BS, G_CHANNEL>(a, stream);
    case G_FULL: return launch_bwd_gate<DT, CPL, BS, G_FULL>(a, stream);
    default: return launch_bwd_gate<DT, CPL, BS, G_TOKEN>(a, stream);   // and without a gate
  }
}

template <int DT>
int sandwich_bwd_rows(SwArgs& a, hipStream_t stream) {
  const Shape s = bwd_shape(a.c.cols);
  a.lpr = s.lpr;
  if (s.bs == 256) return launch_bwd<DT, 1, 256>(a, stream);
  if (s.bs == 512) return launch_bwd<DT, 1, 512>(a, stream);
  return s.cpl == 1 ? launch_bwd<DT, 1, 1024>(a, stream) : launch_bwd<DT, 2, 1024>(a, stream);
}

}  // namespace
