// Balance loss of the router with its counts and gradient: for a sequence of n counted tokens with c_e picks of expert e,
//   L = E sum_e c_e / (K n) P_e,  P_e = mean_t p_te,  p_t = softmax(z_t)
//   dL/dz_te = p_te (v_e - sum_j p_tj v_j),  v_e = E c_e / (K n^2)      (the counts are constants)
// v only enters through differences, so its mean is taken out first: c_e - (sum c) / E is formed from whole numbers, and a
// balanced router's gradient is zero instead of the rounding of two equal terms.
//
// Forward: a block of 4 to 16 waves takes a chunk of tokens and walks through the sequences in it; per sequence, each wave takes
// two to eight tokens at a time (their loads together: a chunk is short, so a row's latency counts), its lanes sum the softmax of
// NE neighbouring experts each in registers, the picks are counted by integer adds in LDS, and the block writes both to slot
// (chunk + sequence) of the workspace: along the tokens either number grows at every step, so slots are distinct and a
// sequence's are consecutive. A second kernel adds a sequence's slots, a fixed set of them per thread in order; a third joins
// the losses where there are several. A short batch of one sequence is one block's, and one launch. Sums have a fixed order,
// integer adds have none that shows: results repeat bit for bit. The forward leaves with every token what the backward needs to
// take it up again (maximum, 1 / sum, sequence or none): one pass over the rows.
#include <algorithm>
#include <type_traits>

#include "../../include/smel_loss.h"
#include "abi_util.h"
#include "common.h"

namespace {

constexpr int MAX_E = 512, MAX_K = 64;

template <int DT>
struct El {
  typedef uint16_t T;
};
template <>
struct El<1> {
  typedef float T;
};
template <int DT>
SMEL_DEV float cvt(typename El<DT>::T b) {
  if constexpr (DT == 1) return b;
  else if constexpr (DT == 0) return __uint_as_float((uint32_t)b << 16);
  else return (float)__builtin_bit_cast(_Float16, b);
}
// N neighbouring values of a row of E from e0 on, `none` past it; one access of element alignment (the hardware takes any address)
template <class T, int N>
struct Run {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V U __attribute__((aligned(sizeof(T))));
};
template <class T>
struct Run<T, 1> {
  typedef T V;
  typedef T U;
};
template <int DT, int N>
SMEL_DEV void ld_run(const typename El<DT>::T* row, int e0, int E, float none, float (&v)[N]) {
  typedef typename El<DT>::T T;
  if constexpr (N > 1) {
    if (e0 + N <= E) {
      const typename Run<T, N>::V q = *(const typename Run<T, N>::U*)(row + e0);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = cvt<DT>(q[i]);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = e0 + i < E ? cvt<DT>(row[e0 + i]) : none;
}
template <int DT, int N>
SMEL_DEV void st_run(typename El<DT>::T* row, int e0, int E, const float (&v)[N]) {
  typedef typename El<DT>::T T;
  T o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (DT == 1) o[i] = v[i];
    else if constexpr (DT == 0) o[i] = f2bf(v[i]);
    else o[i] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);
  }
  if constexpr (N > 1) {
    if (e0 + N <= E) {
      typename Run<T, N>::V q;
#pragma unroll
      for (int i = 0; i < N; ++i) q[i] = o[i];
      *(typename Run<T, N>::U*)(row + e0) = q;
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (e0 + i < E) row[e0 + i] = o[i];
}

// e^x (x <= 0, -inf or NaN) on v_exp_f32: 2^h for h = x log2(e) as rounded, times e^d = 1 + d for what is left, d = x - h ln(2)
// with ln(2) in two parts, so that h's rounding does not grow with |x|. At -inf, or where h overflows to it, d is anything
// finite and the result 0.
SMEL_DEV float exp_acc(float x) {
  const float h = x * 1.4426950408889634f, e = __builtin_amdgcn_exp2f(h);
  const float d = fmaf(-h, -1.9046543e-9f, fmaf(-h, 0.693147182464599609375f, x));
  return fmaf(e, __builtin_amdgcn_fmed3f(d, -1.f, 1.f), e);
}
// 1 / x to its last bits (v_rcp_f32 and one Newton step; x: a row's sum of exponentials, 1 to 512 or NaN)
SMEL_DEV float inverse(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, r, 1.f), r, r);
}

// Sums (or maxima) over the wave of B values at once, uniform. v_permlane32_swap hands two values' halves to each other, so that one
// operation adds both (lanes 0-31: the first's, 32-63: the second's); v_permlane16_swap the same for rows of 16; then four
// rotations within the rows. Four values take 10 operations, not the 24 of one after the other: a short row's share of the
// forward is its instructions (4092 x 256 bf16 in nine sequences: 13 -> 11.3 us; 32768 fp32 rows: 13.4 -> 11.5).
struct Sum {
  SMEL_DEV static float of(float a, float b) { return a + b; }
};
struct Max {
  SMEL_DEV static float of(float a, float b) { return fmaxf(a, b); }
};
template <class Op>
SMEL_DEV float swap32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class Op>
SMEL_DEV float swap16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return Op::of(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <class Op>
SMEL_DEV float rotate16(float v) {   // over a row of 16, in every lane
#define BAL_ROR(n) \
  v = Op::of(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + n, 0xf, 0xf, true)))
  BAL_ROR(8);
  BAL_ROR(4);
  BAL_ROR(2);
  BAL_ROR(1);
#undef BAL_ROR
  return v;
}
// over L lanes (16, 32 or 64), in each of them
template <class Op, int L, int B>
SMEL_DEV void over_lanes(float (&v)[B]) {
  static_assert(L == 16 || B % 2 == 0, "values at once");
  if constexpr (L == 16) {
#pragma unroll
    for (int k = 0; k < B; ++k) v[k] = rotate16<Op>(v[k]);
  } else if constexpr (L == 32) {
#pragma unroll
    for (int k = 0; k < B; k += 2) {   // rows of 16: v[k], v[k + 1], v[k], v[k + 1]
      const uint32_t w = __float_as_uint(rotate16<Op>(swap16<Op>(v[k], v[k + 1])));
      const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
      v[k] = __uint_as_float(r[0]);
      v[k + 1] = __uint_as_float(r[1]);
    }
  } else if constexpr (B == 4) {   // rows of 16: values 0, 2, 1, 3
    const float w = rotate16<Op>(swap16<Op>(swap32<Op>(v[0], v[1]), swap32<Op>(v[2], v[3])));
    v[0] = lane_get(w, 0);
    v[2] = lane_get(w, 16);
    v[1] = lane_get(w, 32);
    v[3] = lane_get(w, 48);
  } else {
    float w = swap32<Op>(v[0], v[1]);
    w = rotate16<Op>(swap16<Op>(w, w));
    v[0] = lane_get(w, 0);
    v[1] = lane_get(w, 32);
  }
}

// A token's experts lie in L lanes, NE to each; a wave takes B runs of 64 / L tokens at a time.
template <int NE_, int L_, int B_>
struct Shape {
  static constexpr int NE = NE_, L = L_, B = B_, RUN = 64 / L, TOKENS = RUN * B;
};

struct Seqs {
  const void* off;   // null: one sequence of all tokens
  int i64;
  int S;
  int64_t T;
  SMEL_DEV int64_t at(int s) const {
    if (!off) return s == 0 ? 0 : T;
    const int64_t v = i64 ? ((const int64_t*)off)[s] : (int64_t)((const int32_t*)off)[s];
    return v < 0 ? 0 : v > T ? T : v;
  }
  // the last s with at(s) <= t, `lo` if there is none after it (empty sequences before the token's own are passed over)
  SMEL_DEV int find(int64_t t, int lo = -1) const {
    int hi = S;   // at(lo) <= t < at(hi + 1)
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (at(m) <= t) lo = m;
      else hi = m;
    }
    return lo;
  }
};

struct Row {      // what the backward takes a token up with
  float m, r;     // its maximum, 1 / its sum of exponentials
  int seq, pad;   // its sequence, -1 where it does not count
};

struct Num {      // of a slot
  int32_t tokens, picks;   // that count (K T < 2^31)
};

struct BalArgs {
  const void* z;
  int64_t ldl, T;
  const void* topi;
  int topi_i64;
  int E, K, chunk;
  const uint8_t* mask;
  Seqs q;
  float coef;
  Row* rows;       // null: no backward
  float* P;        // [slots][E]
  int32_t* C;      // [slots][E]
  Num* N;          // [slots]
  float* loss;
  int64_t* counts;
  float* weights;
  int parts;       // blocks of a sequence's sums
  float* seq_loss; // [S][parts]
  int32_t* seq_n;  // [S]
};

// A sequence's counts and weights of expert x from its picks c and sum P of the softmax, x < E, and the share in the loss of
// the block's experts; `in` counts the sequence's. All threads of the block call it (others with x >= E); the result, of red's
// slot a wave, is thread 0's.
SMEL_DEV float finish_seq(const BalArgs& a, int s, int x, int64_t c, Num in, float P, float* red) {
  const int waves = blockDim.x >> 6;
  const int64_t n = in.tokens;
  float l = 0.f;
  if (x < a.E) {
    const double scale = n > 0 ? (double)a.coef / ((double)a.K * (double)n * (double)n) : 0.0;
    a.counts[(int64_t)s * a.E + x] = c;
    a.weights[(int64_t)s * a.E + x] = (float)((double)(c * a.E - in.picks) * scale);
    l = n > 0 ? (float)((double)(c * a.E) * scale) * P : 0.f;
  }
  l = wave_sum(l);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = l;
  __syncthreads();
  for (int k = 1; k < waves; ++k) l = k == 1 ? red[0] + red[1] : l + red[k];
  return l;
}

// W waves. ONE: all tokens are this block's and one sequence: no slots, the loss at once
template <int DT, class SH, int W, bool ONE>
__global__ __launch_bounds__(64 * W) void bal_fwd_kernel(BalArgs a) {
  typedef typename El<DT>::T T;
  constexpr int NE = SH::NE, L = SH::L, B = SH::B, RUN = SH::RUN;
  __shared__ float sp[W][L * NE];
  __shared__ int sc[MAX_E];
  __shared__ Num sn;
  __shared__ float red[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = lane / L, e0 = lane % L * NE;
  const int64_t c0 = (int64_t)blockIdx.x * a.chunk, c1 = min(c0 + a.chunk, a.T);
  if (a.rows && a.q.off) {   // tokens of no sequence
    for (int64_t t = c0 + threadIdx.x; t < c1; t += 64 * W) a.rows[t].seq = -1;
    __syncthreads();
  }
  int s = ONE ? 0 : max(a.q.find(c0), 0);
  int64_t begin = a.q.at(s), end = a.q.at(s + 1), next;
  for (; s < a.q.S; ++s, begin = end, end = next) {
    const int64_t b = max(begin, c0), e = min(end, c1);
    next = a.q.at(min(s + 2, a.q.S));
    if (!ONE) {
      if (begin >= c1) break;
      if (b >= e) {
        // Two empty ones in a row: on to the last that starts here. Each walked through is a trip to memory (0.2 us): offsets
        // filled up to a fixed length with their last value, three runs of 2^20, took 227 ms, now 10 (the sums' blocks)
        if (s + 1 < a.q.S && next == end) {
          s = a.q.find(end, s + 1) - 1;
          next = a.q.at(s + 2);
        }
        continue;
      }
    }
    for (int i = threadIdx.x; i < a.E; i += 64 * W) sc[i] = 0;
    if (threadIdx.x == 0) sn = Num{0, 0};
    __syncthreads();
    auto pick = [&](int64_t i) -> int64_t {   // pick i of the block's, -1 where it counts nowhere
      if (i >= e * a.K || (a.mask && !a.mask[(uint32_t)i / (uint32_t)a.K])) return -1;   // T K < 2^31
      return a.topi_i64 ? ((const int64_t*)a.topi)[i] : (int64_t)((const int32_t*)a.topi)[i];
    };
    int64_t i0 = b * a.K + threadIdx.x;
    int64_t id = pick(i0);   // on its way while the rows are summed
    float acc[NE];
    int n = 0;
#pragma unroll
    for (int i = 0; i < NE; ++i) acc[i] = 0.f;
    for (int64_t t0 = b + wave * SH::TOKENS + sub; t0 < e + sub; t0 += W * SH::TOKENS) {   // uniform
      float z[B][NE];
      bool keep[B];
#pragma unroll
      for (int k = 0; k < B; ++k) {   // past the end: the last row again, with no share
        const int64_t t = min(t0 + k * RUN, e - 1);
        keep[k] = t0 + k * RUN < e;
        ld_run<DT, NE>((const T*)a.z + t * a.ldl, e0, a.E, -INFINITY, z[k]);
      }
      if (a.mask)
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const bool counts = a.mask[min(t0 + k * RUN, e - 1)];
          keep[k] = keep[k] && counts;
#pragma unroll
          for (int i = 0; i < NE; ++i) z[k][i] = counts ? z[k][i] : 0.f;   // whatever it holds
        }
      float m[B], sum[B];
#pragma unroll
      for (int k = 0; k < B; ++k) {
        m[k] = z[k][0];
#pragma unroll
        for (int i = 1; i < NE; ++i) m[k] = fmaxf(m[k], z[k][i]);
      }
      over_lanes<Max, L>(m);
#pragma unroll
      for (int k = 0; k < B; ++k) {
        sum[k] = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {   // experts past E are at -inf
          z[k][i] = exp_acc(z[k][i] - m[k]);
          sum[k] += z[k][i];
        }
      }
      over_lanes<Sum, L>(sum);
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const float r = inverse(sum[k]), share = keep[k] ? r : 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) acc[i] = fmaf(z[k][i], share, acc[i]);
        n += keep[k];
        if (a.rows && e0 == 0 && t0 + k * RUN < e) a.rows[t0 + k * RUN] = Row{m[k], r, keep[k] ? s : -1, 0};
      }
    }
    int picks = 0;   // the wave's, in its first lane, which leaves the loop last
    while (i0 < e * a.K) {
      const bool in = id >= 0 && id < a.E;
      if (in) atomicAdd(&sc[id], 1);
      picks += __popcll(__ballot(in));
      i0 += 64 * W;
      id = pick(i0);
    }
    if (e0 == 0) atomicAdd(&sn.tokens, n);
    if (lane == 0) atomicAdd(&sn.picks, picks);
#pragma unroll
    for (int i = 0; i < NE; ++i) {   // the wave's runs joined
      if constexpr (L <= 32) acc[i] = swap32<Sum>(acc[i], acc[i]);
      if constexpr (L <= 16) acc[i] = swap16<Sum>(acc[i], acc[i]);
      if (sub == 0) sp[wave][e0 + i] = acc[i];
    }
    __syncthreads();
    auto share = [&](int x) {
      float P = sp[0][x];
#pragma unroll
      for (int k = 1; k < W; ++k) P += sp[k][x];
      return P;
    };
    if constexpr (ONE) {
      const int x = threadIdx.x;
      const float l = finish_seq(a, 0, x, x < a.E ? sc[x] : 0, sn, x < a.E ? share(x) : 0.f, red);
      if (x == 0) {
        *a.loss = l;
        a.weights[a.E] = 1.f;
      }
      return;
    }
    const int64_t slot = (int64_t)blockIdx.x + s;
    for (int x = threadIdx.x; x < a.E; x += 64 * W) {
      a.P[slot * a.E + x] = share(x);
      a.C[slot * a.E + x] = sc[x];
    }
    if (threadIdx.x == 0) a.N[slot] = sn;
    __syncthreads();
  }
}

// A sequence's `1 << lgc` experts: its slots' sums, counts, weights and loss. The block's groups of as many threads take every
// group-th slot each.
template <int BS>
__global__ __launch_bounds__(BS) void bal_seq_kernel(BalArgs a, int lgc) {
  __shared__ float sp[BS], red[BS / 64];
  __shared__ int sc[BS];
  __shared__ Num sn;
  const int s = blockIdx.x / a.parts, part = blockIdx.x % a.parts;
  const int64_t b = a.q.at(s), e = a.q.at(s + 1);
  const int cols = 1 << lgc, groups = BS >> lgc, col = threadIdx.x & (cols - 1), g = threadIdx.x >> lgc, x = (part << lgc) + col;
  const int64_t k0 = b / a.chunk + s, k1 = b < e ? (e - 1) / a.chunk + s : k0 - 1;
  float P = 0.f;
  int c = 0;
  constexpr int U = 8;   // slots at a time: each is a round trip to memory
  if (x < a.E)
    for (int64_t k = k0 + g; k <= k1; k += U * groups) {
      float p[U];
      int q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i = min(k + u * groups, k1) * a.E + x;
        p[u] = a.P[i];
        q[u] = a.C[i];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = k + u * groups <= k1;
        P += in ? p[u] : 0.f;
        c += in ? q[u] : 0;
      }
    }
  if (threadIdx.x < 64) {
    Num n{0, 0};
    for (int64_t k = k0 + threadIdx.x; k <= k1; k += 64) {
      const Num v = a.N[k];
      n.tokens += v.tokens;
      n.picks += v.picks;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      n.tokens += __shfl_xor(n.tokens, o, 64);
      n.picks += __shfl_xor(n.picks, o, 64);
    }
    if (threadIdx.x == 0) sn = n;
  }
  sp[threadIdx.x] = P;
  sc[threadIdx.x] = c;
  __syncthreads();
  if (g == 0)
    for (int k = 1; k < groups; ++k) {
      P += sp[(k << lgc) + col];
      c += sc[(k << lgc) + col];
    }
  const float l = finish_seq(a, s, g == 0 ? x : MAX_E, c, sn, P, red);
  if (threadIdx.x == 0) {
    if (a.q.S * a.parts == 1) {
      *a.loss = l;
      a.weights[a.E] = 1.f;
    } else {
      a.seq_loss[blockIdx.x] = l;
      if (part == 0) a.seq_n[s] = sn.tokens > 0;
    }
  }
}

__global__ __launch_bounds__(1024) void bal_join_kernel(BalArgs a) {
  __shared__ float red[16];
  __shared__ int cnt[16];
  float l = 0.f;
  int n = 0;
  for (int s = threadIdx.x; s < a.q.S * a.parts; s += 1024) l += a.seq_loss[s];
  for (int s = threadIdx.x; s < a.q.S; s += 1024) n += a.seq_n[s];
  l = wave_sum(l);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, 64);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6] = l;
    cnt[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 16; ++k) {
      l += red[k];
      n += cnt[k];
    }
    const float r = 1.f / (float)max(n, 1);
    *a.loss = l * r;
    a.weights[(int64_t)a.q.S * a.E] = r;
  }
}

template <int DT, class SH>
__global__ __launch_bounds__(256) void bal_bwd_kernel(BalArgs a, const float* __restrict__ go, void* __restrict__ dz) {
  typedef typename El<DT>::T T;
  constexpr int NE = SH::NE, L = SH::L, B = SH::B, RUN = SH::RUN;
  const int lane = threadIdx.x & 63, e0 = lane % L * NE;
  const int64_t w0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * SH::TOKENS, t0 = w0 + lane / L;
  if (w0 >= a.T) return;
  const float g = *go * a.weights[(int64_t)a.q.S * a.E];
  float z[B][NE], v[B][NE];
  Row row[B];
#pragma unroll
  for (int k = 0; k < B; ++k) {
    const int64_t t = min(t0 + k * RUN, a.T - 1);
    row[k] = a.rows[t];
    ld_run<DT, NE>((const T*)a.z + t * a.ldl, e0, a.E, -INFINITY, z[k]);
  }
  if (a.q.S == 1) {
    ld_run<1, NE>(a.weights, e0, a.E, 0.f, v[0]);
#pragma unroll
    for (int k = 1; k < B; ++k)
#pragma unroll
      for (int i = 0; i < NE; ++i) v[k][i] = v[0][i];
  } else {
#pragma unroll
    for (int k = 0; k < B; ++k) ld_run<1, NE>(a.weights + (int64_t)max(row[k].seq, 0) * a.E, e0, a.E, 0.f, v[k]);
  }
  float dot[B];
#pragma unroll
  for (int k = 0; k < B; ++k) {
    dot[k] = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {   // past E: p = 0
      z[k][i] = exp_acc(z[k][i] - row[k].m) * row[k].r;
      dot[k] = fmaf(z[k][i], v[k][i], dot[k]);
    }
  }
  over_lanes<Sum, L>(dot);
#pragma unroll
  for (int k = 0; k < B; ++k) {
    if (t0 + k * RUN >= a.T) break;
    float d[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) d[i] = row[k].seq >= 0 ? g * (z[k][i] * (v[k][i] - dot[k])) : 0.f;
    st_run<DT, NE>((T*)dz + (t0 + k * RUN) * a.E, e0, a.E, d);
  }
}

// ------------------------------------------------------------------------------------------------ host

// Sequences of under 64 tokens on average: blocks of four waves and about four sequences (each costs a block a few round
// trips to memory, so many blocks have to be under way: 131072 tokens in 4096 sequences 129 -> 40 us).
bool short_seqs(int64_t T, int64_t S) { return S > 1 && S * 64 > T; }
// To 2048 tokens on average: eight waves and chunks of 32, twice the blocks; a sequence's slots are few (517 x 256 bf16, with the
// slots' sums: 9.9 -> 8.8 us; 4092 in nine sequences 16.9 -> 16.2; 8192 x 256 fp32 in 64: 23 -> 18, in one 11.9 -> 12.9)
bool medium_seqs(int64_t T, int64_t S) { return T <= S * 2048; }
// tokens of a forward block: up to 512 blocks, 256 of sixteen waves, four tokens for a wave at least
int chunk_of(int64_t T, int64_t S) {
  if (short_seqs(T, S)) return (int)std::max<int64_t>(4, 4 * T / S);
  if (medium_seqs(T, S)) return (int)std::max<int64_t>((T + 511) / 512, 32);
  return (int)std::max<int64_t>((T + 255) / 256, 64);
}
int64_t chunks_of(int64_t T, int64_t S) { return T ? (T + chunk_of(T, S) - 1) / chunk_of(T, S) : 0; }
constexpr int64_t ONE_BLOCK = 192;   // tokens of one sequence that a block takes alone

// Blocks of a sequence's sums: one, or where its slots are many, one for each 64 experts (256 slots of 512 experts: 19 us by one
// CU, 6 by eight with 2 for the join; of 256: 10.2, or 5.7 and 2).
int parts_of(int64_t T, int64_t E, int64_t S) {
  return (chunks_of(T, S) + S) / S * E >= 1 << 16 ? (int)((E + 63) / 64) : 1;
}

struct Ws {
  int64_t P, C, N, loss, n, bytes;
};
Ws ws_of(int64_t T, int64_t E, int64_t S) {
  auto up = [](int64_t b) { return (b + 15) / 16 * 16; };
  const int64_t slots = chunks_of(T, S) + S;
  Ws w;
  w.P = 0;
  w.C = up(slots * E * 4);
  w.N = w.C + up(slots * E * 4);
  w.loss = w.N + up(slots * 8);
  w.n = w.loss + up(S * parts_of(T, E, S) * 4);
  w.bytes = w.n + up(S * 4);
  return w;
}

int check(const char* name, const void* z, int64_t ldl, int dtype, int64_t T, int64_t E, int64_t S, const void* off) {
  SMEL_REQUIRE(T >= 0 && T <= (int64_t)1 << 24, SMEL_EUNSUPPORTED, "%s: T=%lld tokens, 0 to 2^24", name, (long long)T);
  SMEL_REQUIRE(E >= 1 && E <= MAX_E, SMEL_EUNSUPPORTED, "%s: E=%lld experts, 1 to %d", name, (long long)E, MAX_E);
  SMEL_REQUIRE(S >= 1 && S <= (int64_t)1 << 22, SMEL_EUNSUPPORTED, "%s: S=%lld sequences, 1 to 2^22", name, (long long)S);
  SMEL_REQUIRE(off || S == 1, SMEL_EINVAL, "%s: %lld sequences without offsets", name, (long long)S);
  SMEL_REQUIRE(dtype >= 0 && dtype <= 2, SMEL_EINVAL, "%s: dtype %d (0 = bf16, 1 = fp32, 2 = fp16)", name, dtype);
  SMEL_REQUIRE(T == 0 || z, SMEL_EINVAL, "%s: null logits", name);
  SMEL_REQUIRE(T <= 1 || ldl >= E, SMEL_EINVAL, "%s: row stride %lld < E=%lld", name, (long long)ldl, (long long)E);
  return 0;
}

template <int V>
struct Int {
  static constexpr int value = V;
};
// f(dtype, shape) as constants: 16 bytes of a row to a lane, 16 lanes at least (131072 x 64 bf16, forward: 12 us, 64 lanes of an
// expert each 21; 4092 x 256 in nine sequences: 9.7, 64 lanes of four 10.4; 32768 x 256 fp32 backward: 64 lanes of four 11.6,
// 32 of eight 14); two or four rows' loads at a time (131072 x 64 in 4096 sequences: 33 us with two, 42 with four)
template <class F>
void pick(int dtype, int64_t E, F f) {
  auto by_e = [&](auto dt) {
    constexpr bool f32 = decltype(dt)::value == 1;
    if (E <= 64) f(dt, Shape<4, 16, 2>{});
    else if (E <= 128) f(dt, std::conditional_t<f32, Shape<4, 32, 4>, Shape<8, 16, 2>>{});
    else if (E <= 256) f(dt, std::conditional_t<f32, Shape<4, 64, 4>, Shape<8, 32, 2>>{});
    else f(dt, Shape<8, 64, 2>{});
  };
  if (dtype == 0) by_e(Int<0>{});
  else if (dtype == 1) by_e(Int<1>{});
  else by_e(Int<2>{});
}

}  // namespace

extern "C" int64_t smel_balance_ws_bytes(int64_t T, int64_t E, int64_t S) {
  if (T < 0 || E < 1 || E > MAX_E || S < 1) return 0;
  return ws_of(T, E, S).bytes;
}

extern "C" int smel_balance_fwd(const void* logits, int64_t ldl, int32_t dtype, const void* topi, int32_t topi_i64,
                                int64_t T, int64_t E, int64_t K, const uint8_t* mask, const void* offsets,
                                int32_t off_i64, int64_t S, float coef, float* loss, int64_t* counts, float* row_stats,
                                float* weights, void* ws, int64_t ws_bytes, hipStream_t stream) {
  const int rc = check("balance_fwd", logits, ldl, dtype, T, E, S, offsets);
  if (rc) return rc;
  SMEL_REQUIRE(K >= 1 && K <= MAX_K, SMEL_EUNSUPPORTED, "balance_fwd: K=%lld, 1 to %d", (long long)K, MAX_K);
  SMEL_REQUIRE((T == 0 || topi) && loss && counts && weights, SMEL_EINVAL, "balance_fwd: null pointer");
  const Ws w = ws_of(T, E, S);
  SMEL_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= w.bytes, SMEL_EINVAL,
               "balance_fwd: a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)w.bytes,
               (long long)ws_bytes);
  SMEL_REQUIRE((uintptr_t)row_stats % 16 == 0, SMEL_EINVAL, "balance_fwd: row_stats must be 16-byte aligned");
  char* const base = (char*)ws;
  BalArgs a{};
  a.z = logits;
  a.ldl = ldl;
  a.T = T;
  a.topi = topi;
  a.topi_i64 = topi_i64;
  a.E = (int)E;
  a.K = (int)K;
  a.mask = mask;
  a.q = Seqs{offsets, off_i64, (int)S, T};
  a.coef = coef;
  a.rows = (Row*)row_stats;
  a.loss = loss;
  a.counts = counts;
  a.weights = weights;
  if (S == 1 && T <= ONE_BLOCK) {
    a.chunk = ONE_BLOCK;
    pick(dtype, E, [&](auto dt, auto sh) {
      bal_fwd_kernel<decltype(dt)::value, decltype(sh), 16, true><<<1, 1024, 0, stream>>>(a);
    });
    return smel::launch_status();
  }
  a.chunk = chunk_of(T, S);
  a.P = (float*)(base + w.P);
  a.C = (int32_t*)(base + w.C);
  a.N = (Num*)(base + w.N);
  a.parts = parts_of(T, E, S);
  a.seq_loss = (float*)(base + w.loss);
  a.seq_n = (int32_t*)(base + w.n);
  if (T)
    pick(dtype, E, [&](auto dt, auto sh) {
      constexpr int d = decltype(dt)::value;
      typedef decltype(sh) SH;
      const unsigned n = (unsigned)chunks_of(T, S);
      if (short_seqs(T, S)) bal_fwd_kernel<d, SH, 4, false><<<n, 256, 0, stream>>>(a);
      else if (medium_seqs(T, S)) bal_fwd_kernel<d, SH, 8, false><<<n, 512, 0, stream>>>(a);
      else bal_fwd_kernel<d, SH, 16, false><<<n, 1024, 0, stream>>>(a);
    });
  int lgc = 6;
  while (a.parts == 1 && (1 << lgc) < E) ++lgc;
  const unsigned n = (unsigned)(S * a.parts);
  if (n <= 512) bal_seq_kernel<1024><<<n, 1024, 0, stream>>>(a, lgc);
  else bal_seq_kernel<512><<<n, 512, 0, stream>>>(a, lgc);
  if (n > 1) bal_join_kernel<<<1, 1024, 0, stream>>>(a);
  return smel::launch_status();
}

extern "C" int smel_balance_bwd(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E, int64_t S,
                                const float* row_stats, const float* weights, const float* go, void* dlogits,
                                hipStream_t stream) {
  const int rc = check("balance_bwd", logits, ldl, dtype, T, E, S, weights);
  if (rc) return rc;
  if (T == 0) return 0;
  SMEL_REQUIRE(row_stats && weights && go && dlogits, SMEL_EINVAL, "balance_bwd: null pointer");
  SMEL_REQUIRE((uintptr_t)row_stats % 16 == 0, SMEL_EINVAL, "balance_bwd: row_stats must be 16-byte aligned");
  BalArgs a{};
  a.z = logits;
  a.ldl = ldl;
  a.T = T;
  a.E = (int)E;
  a.q = Seqs{nullptr, 0, (int)S, T};
  a.rows = (Row*)const_cast<float*>(row_stats);
  a.weights = const_cast<float*>(weights);
  pick(dtype, E, [&](auto dt, auto sh) {
    typedef decltype(sh) SH;
    constexpr int tokens = 4 * SH::TOKENS;
    bal_bwd_kernel<decltype(dt)::value, SH><<<(unsigned)((T + tokens - 1) / tokens), 256, 0, stream>>>(a, go, dlogits);
  });
  return smel::launch_status();
}
