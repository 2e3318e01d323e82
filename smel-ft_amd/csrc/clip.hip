// The global norm of many tensors, and every tensor scaled by min(1, max_norm / (norm + eps)).
//
// The tensors travel as kernel arguments, a table a launch; a block takes chunks of their values, wherever they lie in the list. Squares
// are summed in 64 bits: no value of 32 bits over- or underflows there, and the sum of 2^28 squares keeps its last fp32 bit. A block's
// sum goes to the workspace, and whoever needs the norm adds those in order: no atomics, the same bits every time.
// HBM-bound: 2^28 bf16 values 94 us for the norm (5.7 TB/s) and 200 for the scaling (5.4); a LoRA layer's twelve tensors 4.3 and 5.8,
// where both are a launch's latency.
#include <stdlib.h>

#include <algorithm>

#include "../../include/smel_clip.h"
#include "abi_util.h"
#include "common.h"
#include "rows.h"

namespace {

constexpr int MAX_JOBS = 120;      // of one launch: 32 bytes each of the 4 KiB of kernel arguments
constexpr int CHUNK = 8192;        // values of a block's turn
constexpr int64_t MOST_BLOCKS = 2048;   // of one launch

struct Entry {
  const void* in;
  void* out;
  int64_t n;
  uint32_t first, dtype;   // the first of its chunks in the launch
};
struct Jobs {
  int32_t n;
  uint32_t chunks;
  Entry e[MAX_JOBS];
};

// dtype of the interface (0 bf16, 1 fp32, 2 fp16) as rows.h numbers them
constexpr int ROWS_TYPE[3] = {0, 2, 1};

// f(type, entry, first value, values) for each chunk of the block
template <typename F>
SMEL_DEV void each_chunk(const Jobs& js, F f) {
  for (uint32_t c = blockIdx.x; c < js.chunks; c += gridDim.x) {
    int lo = 0, hi = js.n - 1;   // the last entry whose first chunk is at most c
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (js.e[mid].first <= c) lo = mid;
      else hi = mid - 1;
    }
    const Entry& e = js.e[lo];
    const int64_t at = (int64_t)(c - e.first) * CHUNK;
    const int64_t left = e.n - at;
    f(e, at, (int)(left < CHUNK ? left : CHUNK));
  }
}

// A chunk's values in registers, all of them on their way at once: thread i has the 8 from 8 i on, 8 (256 + i) on, .... Zeros behind n.
constexpr int TURNS = CHUNK / (8 * 256);
template <int DT>
struct Chunk {
  Raw<DT> r[TURNS];
  SMEL_DEV void load(const void* in, int64_t at, int n) {
    const typename El<DT>::T* const p = (const typename El<DT>::T*)in + at;
#pragma unroll
    for (int k = 0; k < TURNS; ++k) {
      const int e = 8 * (256 * k + (int)threadIdx.x);
      r[k] = Raw<DT>{};
      if (e < n) r[k] = load8<DT>(p, e, n);
    }
  }
};
template <int DT>
SMEL_DEV double squares(const void* in, int64_t at, int n) {
  Chunk<DT> c;
  c.load(in, at, n);
  double v = 0;
#pragma unroll
  for (int k = 0; k < TURNS; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) v = __builtin_fma((double)c.r[k].at(j), (double)c.r[k].at(j), v);
  return v;
}
template <int DT>
SMEL_DEV uint32_t largest(const void* in, int64_t at, int n) {   // bits of |x|: NaN is above infinity
  Chunk<DT> c;
  c.load(in, at, n);
  uint32_t v = 0;
#pragma unroll
  for (int k = 0; k < TURNS; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) v = max(v, __float_as_uint(fabsf(c.r[k].at(j))));
  return v;
}

template <bool INF>
SMEL_DEV double joined(double a, double b) {
  return INF ? (b > a || b != b ? b : a) : a + b;     // the largest, NaN above all; or the sum
}
// of the 256 threads' v, in a fixed order, for all of them
template <bool INF>
SMEL_DEV double block_total(double v, double* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = joined<INF>(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return joined<INF>(joined<INF>(red[0], red[1]), joined<INF>(red[2], red[3]));
}

template <bool INF>
__global__ __launch_bounds__(256) void norm_parts_kernel(Jobs js, double* __restrict__ part) {
  __shared__ double red[4];
  double v = 0;
  uint32_t m = 0;
  each_chunk(js, [&](const Entry& e, int64_t at, int n) {
    if constexpr (INF)
      m = max(m, e.dtype == 0 ? largest<0>(e.in, at, n) : e.dtype == 1 ? largest<2>(e.in, at, n) : largest<1>(e.in, at, n));
    else
      v += e.dtype == 0 ? squares<0>(e.in, at, n) : e.dtype == 1 ? squares<2>(e.in, at, n) : squares<1>(e.in, at, n);
  });
  if constexpr (INF) v = (double)__uint_as_float(m);
  v = block_total<INF>(v, red);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// the parts [n] as one, eight loads at a time
template <bool INF>
SMEL_DEV double parts_total(const double* __restrict__ part, int n, double* red) {
  double v = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += 256) v = joined<INF>(v, part[i]);
  return block_total<INF>(v, red);
}
// one part of many, or (norm given) the norm itself
template <bool INF>
__global__ __launch_bounds__(256) void norm_total_kernel(const double* __restrict__ part, int n, double* __restrict__ total,
                                                         float* __restrict__ norm) {
  __shared__ double red[4];
  const double v = parts_total<INF>(part, n, red);
  if (threadIdx.x != 0) return;
  if (norm) *norm = (float)(INF ? v : sqrt(v));
  else *total = v;
}

template <int DT>
SMEL_DEV void scaled(const Entry& en, int64_t at, int n, float c) {
  typedef typename El<DT>::T T;
  T* const o = (T*)en.out + at;
  Chunk<DT> x;
  x.load(en.in, at, n);
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int e = 8 * (256 * k + (int)threadIdx.x);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x.r[k].at(j) * c;
    x.r[k].set(v);
    if (e < n) store8<DT>(o, e, n, x.r[k]);
  }
}
// Every block adds up the parts itself (a few kilobytes from the L2): a launch less, and no wait for it
template <bool INF>
__global__ __launch_bounds__(256) void scale_kernel(Jobs js, const double* __restrict__ part, int n_parts, double max_norm, double eps,
                                                    float* __restrict__ norm) {
  __shared__ double red[4];
  double v = parts_total<INF>(part, n_parts, red);
  if (!INF) v = sqrt(v);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)v;
  const double f = max_norm / (v + eps);
  const float c = f >= 1.0 ? 1.f : (float)f;     // NaN stays
  each_chunk(js, [&](const Entry& e, int64_t at, int n) {
    if (c == 1.f && e.in == e.out) return;
    if (e.dtype == 0) scaled<0>(e, at, n, c);
    else if (e.dtype == 1) scaled<2>(e, at, n, c);
    else scaled<1>(e, at, n, c);
  });
}

// ------------------------------------------------------------------------------------------------ host

constexpr int64_t SIZE[3] = {2, 4, 2};

int check(const char* name, const smel_clip_job* jobs, int32_t n) {
  SMEL_REQUIRE(n >= 0 && (jobs || n == 0), SMEL_EINVAL, "%s: null jobs", name);
  for (int32_t k = 0; k < n; ++k) {
    const smel_clip_job& j = jobs[k];
    SMEL_REQUIRE(j.n >= 0 && j.dtype >= 0 && j.dtype <= 2, SMEL_EINVAL, "%s: job %d: %lld values of dtype %lld (0 bf16, 1 fp32, 2 fp16)",
                 name, k, (long long)j.n, (long long)j.dtype);
    SMEL_REQUIRE(j.n < (int64_t)1 << 40, SMEL_EUNSUPPORTED, "%s: job %d: %lld values", name, k, (long long)j.n);
    SMEL_REQUIRE(j.n == 0 || (j.in && (uintptr_t)j.in % SIZE[j.dtype] == 0), SMEL_EINVAL, "%s: job %d: null or unaligned values", name, k);
  }
  return 0;
}

struct Range {
  uintptr_t lo, hi;
  bool out;
};
// Nothing that is written may be read or written by another job
int apart(const smel_clip_job* jobs, int32_t n) {
  Range* const r = (Range*)malloc(sizeof(Range) * 2 * (n > 0 ? n : 1));
  SMEL_REQUIRE(r, SMEL_EINVAL, "clip_grads: no host memory");
  int64_t m = 0;
  bool ok = true;
  for (int32_t k = 0; k < n; ++k) {
    const smel_clip_job& j = jobs[k];
    if (j.n == 0) continue;
    const uintptr_t bytes = (uintptr_t)(j.n * SIZE[j.dtype]);
    ok = ok && j.out && (uintptr_t)j.out % SIZE[j.dtype] == 0;
    r[m++] = Range{(uintptr_t)j.out, (uintptr_t)j.out + bytes, true};
    if (j.in != j.out) r[m++] = Range{(uintptr_t)j.in, (uintptr_t)j.in + bytes, false};
  }
  std::sort(r, r + m, [](const Range& a, const Range& b) { return a.lo < b.lo; });
  uintptr_t read = 0, written = 0;   // the ends of what lies before
  bool clear = true;
  for (int64_t i = 0; i < m; ++i) {
    if (r[i].lo < written || (r[i].out && r[i].lo < read)) clear = false;
    uintptr_t& end = r[i].out ? written : read;
    end = end > r[i].hi ? end : r[i].hi;
  }
  free(r);
  SMEL_REQUIRE(ok, SMEL_EINVAL, "clip_grads: null or unaligned output");
  SMEL_REQUIRE(clear, SMEL_EINVAL, "clip_grads: an output overlaps another tensor of the call");
  return 0;
}

// the next launch's table from job `at` (value `from` of it) on
struct Cursor {
  int32_t job;
  int64_t from;
};
Cursor fill(const smel_clip_job* jobs, int32_t n, Cursor at, Jobs& js) {
  constexpr int64_t MOST_CHUNKS = (int64_t)1 << 31;
  js.n = 0;
  int64_t chunks = 0;
  while (at.job < n && js.n < MAX_JOBS && chunks < MOST_CHUNKS) {
    const smel_clip_job& j = jobs[at.job];
    int64_t left = j.n - at.from;
    if (left > 0) {
      int64_t c = (left + CHUNK - 1) / CHUNK;
      if (c > MOST_CHUNKS - chunks) {
        c = MOST_CHUNKS - chunks;
        left = c * CHUNK;
      }
      const int64_t off = at.from * SIZE[j.dtype];
      js.e[js.n++] = Entry{(const char*)j.in + off, (char*)j.out + off, left, (uint32_t)chunks, (uint32_t)j.dtype};
      chunks += c;
    }
    at.from += left;
    if (at.from >= j.n) at = Cursor{at.job + 1, 0};
  }
  js.chunks = (uint32_t)chunks;
  return at;
}
int64_t blocks_of(const Jobs& js) { return js.chunks < MOST_BLOCKS ? js.chunks : MOST_BLOCKS; }

template <typename F>
int each(const smel_clip_job* jobs, int32_t n, F f) {
  Jobs js;
  for (Cursor at{0, 0}; at.job < n;) {
    at = fill(jobs, n, at, js);
    if (js.n == 0) break;
    const int rc = f(js);
    if (rc) return rc;
  }
  return 0;
}

int parts_launches(const char* name, const smel_clip_job* jobs, int32_t n, int32_t type, float* norm, void* ws, int64_t ws_bytes,
                   int64_t& parts, hipStream_t stream) {
  SMEL_REQUIRE(type == 0 || type == 1, SMEL_EINVAL, "%s: norm type %d (0 = 2-norm, 1 = largest magnitude)", name, type);
  SMEL_REQUIRE(norm, SMEL_EINVAL, "%s: null pointer", name);
  const int64_t need = smel_clip_ws(jobs, n);
  SMEL_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, SMEL_EINVAL,
               "%s: an aligned workspace of %lld bytes is needed (got %lld)", name, (long long)need, (long long)ws_bytes);
  double* const part = (double*)ws;
  parts = 0;
  return each(jobs, n, [&](const Jobs& js) {
    const int64_t b = blocks_of(js);
    if (type) norm_parts_kernel<true><<<(unsigned)b, 256, 0, stream>>>(js, part + parts);
    else norm_parts_kernel<false><<<(unsigned)b, 256, 0, stream>>>(js, part + parts);
    parts += b;
    return smel::launch_status();
  });
}
int total_launch(int32_t type, const double* part, int64_t parts, double* total, float* norm, hipStream_t stream) {
  if (type) norm_total_kernel<true><<<1, 256, 0, stream>>>(part, (int)parts, total, norm);
  else norm_total_kernel<false><<<1, 256, 0, stream>>>(part, (int)parts, total, norm);
  return smel::launch_status();
}

}  // namespace

extern "C" int64_t smel_clip_ws(const smel_clip_job* jobs, int32_t n_jobs) {
  if (check("clip", jobs, n_jobs)) return -1;
  int64_t parts = 0;
  each(jobs, n_jobs, [&](const Jobs& js) {
    parts += blocks_of(js);
    return 0;
  });
  return 8 * (parts + 1);
}

extern "C" int smel_grad_norm(const smel_clip_job* jobs, int32_t n_jobs, int32_t norm_type, float* norm, void* ws, int64_t ws_bytes,
                              hipStream_t stream) {
  const int rc = check("grad_norm", jobs, n_jobs);
  if (rc) return rc;
  int64_t parts;
  const int rl = parts_launches("grad_norm", jobs, n_jobs, norm_type, norm, ws, ws_bytes, parts, stream);
  return rl ? rl : total_launch(norm_type, (double*)ws, parts, nullptr, norm, stream);
}

extern "C" int smel_clip_grads(const smel_clip_job* jobs, int32_t n_jobs, int32_t norm_type, double max_norm, double eps, float* norm,
                               void* ws, int64_t ws_bytes, hipStream_t stream) {
  int rc = check("clip_grads", jobs, n_jobs);
  if (rc) return rc;
  SMEL_REQUIRE(max_norm >= 0 && eps >= 0, SMEL_EINVAL, "clip_grads: max_norm %g and eps %g must not be negative", max_norm, eps);
  rc = apart(jobs, n_jobs);
  if (rc) return rc;
  int64_t parts;
  rc = parts_launches("clip_grads", jobs, n_jobs, norm_type, norm, ws, ws_bytes, parts, stream);
  if (rc) return rc;
  double* part = (double*)ws;
  int64_t n_parts = parts;
  if (parts == 0 || parts > 4 * MOST_BLOCKS) {   // nothing to scale, or more than every block should read
    rc = total_launch(norm_type, part, parts, part + parts, parts ? nullptr : norm, stream);
    if (rc) return rc;
    part += parts;
    n_parts = 1;
  }
  float* to = norm;     // of the first launch
  return each(jobs, n_jobs, [&](const Jobs& js) {
    const unsigned b = (unsigned)blocks_of(js);
    if (norm_type) scale_kernel<true><<<b, 256, 0, stream>>>(js, part, (int)n_parts, max_norm, eps, to);
    else scale_kernel<false><<<b, 256, 0, stream>>>(js, part, (int)n_parts, max_norm, eps, to);
    to = nullptr;
    return smel::launch_status();
  });
}
