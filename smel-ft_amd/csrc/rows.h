// Rows of bf16, fp16 or fp32 values in chunks of 8, at any element alignment: loads, stores, conversions, and sums over the
// threads of a row (shared by the row kernels with trained weights).
#pragma once
#include "common.h"

namespace {

// storage types: 0 = bf16, 1 = fp16, 2 = fp32
template <int DT>
struct El {
  typedef uint16_t T;
};
template <>
struct El<2> {
  typedef float T;
};
typedef u32x4_t __attribute__((aligned(2))) u32x4_a2;
typedef f32x4_t __attribute__((aligned(4))) f32x4_a4;

template <int DT>
SMEL_DEV float cvt(uint32_t b) {
  if constexpr (DT == 0)
    return __uint_as_float(b << 16);
  else
    return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
template <int DT>
SMEL_DEV uint32_t enc(float f) {
  if constexpr (DT == 0)
    return f2bf(f);
  else
    return __builtin_bit_cast(uint16_t, (_Float16)f);
}
template <int DT>
SMEL_DEV float round_to(float f) {
  if constexpr (DT == 2)
    return f;
  else
    return cvt<DT>(enc<DT>(f));
}

// 8 elements as stored
template <int DT>
struct Raw {
  u32x4_t q[DT == 2 ? 2 : 1];
  SMEL_DEV float at(int j) const {
    if constexpr (DT == 2)
      return __uint_as_float(q[j >> 2][j & 3]);
    else
      return cvt<DT>((j & 1) ? q[0][j >> 1] >> 16 : q[0][j >> 1] & 0xffffu);
  }
  SMEL_DEV void set(const float v[8]) {
    if constexpr (DT == 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j >> 2][j & 3] = __float_as_uint(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[0][j] = enc<DT>(v[2 * j]) | enc<DT>(v[2 * j + 1]) << 16;
    }
  }
};
// 8 elements of a row of n from e0 (< n) on, zero past the row
template <int DT>
SMEL_DEV Raw<DT> load8(const typename El<DT>::T* p, int e0, int n) {
  Raw<DT> r;
  if (e0 + 8 <= n) {
    if constexpr (DT == 2) {
      const f32x4_a4* f = (const f32x4_a4*)(p + e0);
      r.q[0] = __builtin_bit_cast(u32x4_t, (f32x4_t)f[0]);
      r.q[1] = __builtin_bit_cast(u32x4_t, (f32x4_t)f[1]);
    } else {
      r.q[0] = *(const u32x4_a2*)(p + e0);
    }
    return r;
  }
  if constexpr (DT == 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r.q[j >> 2][j & 3] = e0 + j < n ? __float_as_uint(p[e0 + j]) : 0u;
  } else {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = e0 + j < n ? p[e0 + j] : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.q[0][j] = v[2 * j] | v[2 * j + 1] << 16;
  }
  return r;
}
// Nontemporal: the rows written are more than an L2 holds, and what is read again is the rows (32749 x 2048 bf16: forward 57.9 ->
// 56.7 us, backward 92.6 -> 87.2; 4092 x 2048 with the add: 15.3 -> 14.4 and 18.9 -> 18.7). KEEP: what the next kernel reads, the weights' sums
template <int DT, bool KEEP = false>
SMEL_DEV void store8(typename El<DT>::T* p, int e0, int n, const Raw<DT>& r) {
  if (e0 + 8 <= n) {
    if constexpr (DT == 2) {
      f32x4_a4* f = (f32x4_a4*)(p + e0);
      if constexpr (KEEP) {
        f[0] = __builtin_bit_cast(f32x4_t, r.q[0]);
        f[1] = __builtin_bit_cast(f32x4_t, r.q[1]);
      } else {
        __builtin_nontemporal_store(__builtin_bit_cast(f32x4_t, r.q[0]), f);
        __builtin_nontemporal_store(__builtin_bit_cast(f32x4_t, r.q[1]), f + 1);
      }
    } else {
      __builtin_nontemporal_store(r.q[0], (u32x4_a2*)(p + e0));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (e0 + j < n) {
      if constexpr (DT == 2)
        p[e0 + j] = __uint_as_float(r.q[j >> 2][j & 3]);
      else
        p[e0 + j] = (uint16_t)((j & 1) ? r.q[0][j >> 1] >> 16 : r.q[0][j >> 1]);
    }
}

// w or b of a chunk; `one` where there is none
template <int WT>
SMEL_DEV void weight8(const void* p, int e0, int n, float one, float v[8]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = one;
    return;
  }
  const Raw<WT> r = load8<WT>((const typename El<WT>::T*)p, e0, n);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = r.at(j);
}

// sums over the lpr threads of a row: xor butterfly over its lanes, then the row's waves in order. red: 16 floats a value. lpr is a
// power of two, or the whole block's threads (ONE: its only row)
template <int N, bool ONE = false>
SMEL_DEV void row_sums(float (&v)[N], int lpr, float* red) {
  for (int o = 1; o < lpr && o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o, 64);
  if (lpr > 64) {
    const int wave = threadIdx.x >> 6, nw = lpr >> 6, w0 = ONE ? 0 : wave & ~(nw - 1);
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) red[i * 16 + wave] = v[i];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[i * 16 + w0];
      for (int k = 1; k < nw; ++k) v[i] += red[i * 16 + w0 + k];
    }
  }
}

}  // namespace
