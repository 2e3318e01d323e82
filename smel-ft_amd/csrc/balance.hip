// Balance loss of the router with its counts and gradient: for a sequence of n counted tokens with c_e picks of expert e,
//   L = E sum_e c_e / (K n) P_e,  P_e = mean_t p_te,  p_t = softmax(z_t)
//   dL/dz_te = p_te (v_e - sum_j p_tj v_j),  v_e = E c_e / (K n^2)      (the counts are constants)
// v only enters through differences, so its mean is taken out first: c_e - (sum c) / E is formed from whole numbers, and a
// balanced router's gradient is zero instead of the rounding of two equal terms.
//
// Forward: a block of 16 waves takes a chunk of tokens and walks through the sequences in it; per sequence, each wave takes four
// tokens at a time (their loads together: a chunk is short, so a row's latency counts), its lanes sum the softmax of NE
// neighbouring experts each in registers, the picks are counted by integer adds in LDS, and the block writes both to slot
// (chunk + sequence) of the workspace: along the tokens either number grows at every step, so slots are distinct and a
// sequence's are consecutive. A second kernel (a block per sequence) adds a sequence's slots, a fixed set of them per thread in
// order; a third joins the sequences' losses where there are several. A short batch of one sequence is one block's, and one
// launch. Sums have a fixed order, integer adds have none that shows: results repeat bit for bit. The forward leaves with every
// token what the backward needs to take it up again (maximum, 1 / sum, sequence or none): one pass, four rows a wave.
#include <algorithm>

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
template <class Op, int B>
SMEL_DEV void over_wave(float (&v)[B]) {
  static_assert(B == 2 || B == 4, "values at once");
  if constexpr (B == 4) {   // rows of 16: values 0, 2, 1, 3
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
  // the last s with at(s) <= t, or -1 (empty sequences before the token's own are passed over)
  SMEL_DEV int find(int64_t t) const {
    int lo = -1, hi = S;   // at(lo) <= t < at(hi + 1)
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
  int32_t* N;      // [slots] counted tokens
  float* loss;
  int64_t* counts;
  float* weights;
  float* seq_loss; // [S]
  int32_t* seq_n;  // [S]
};

template <int NE>
constexpr int TB = NE == 8 ? 2 : 4;   // tokens of a wave at a time

// A sequence's counts, weights and loss from expert x's picks c and sum P of the softmax, x < E in thread x; the sums over
// the experts go through red and tot (a slot a wave). All threads of the block call it; the result is thread 0's.
SMEL_DEV float finish_seq(const BalArgs& a, int s, int x, int64_t c, int64_t n, float P, float* red, long long* tot) {
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
  const bool mine = x < a.E;
  if (mine) a.counts[(int64_t)s * a.E + x] = c;
  long long ct = mine ? c : 0;   // picks in range, over all experts
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) ct += __shfl_xor(ct, o, 64);
  if ((threadIdx.x & 63) == 0) tot[wave] = ct;
  __syncthreads();
  ct = 0;
  for (int k = 0; k < waves; ++k) ct += tot[k];
  float l = 0.f;
  if (mine) {
    const double scale = n > 0 ? (double)a.coef / ((double)a.K * (double)n * (double)n) : 0.0;
    a.weights[(int64_t)s * a.E + x] = (float)((double)(c * a.E - ct) * scale);
    l = n > 0 ? (float)((double)(c * a.E) * scale) * P : 0.f;
  }
  l = wave_sum(l);
  if ((threadIdx.x & 63) == 0) red[wave] = l;
  __syncthreads();
  for (int k = 1; k < waves; ++k) l = k == 1 ? red[0] + red[1] : l + red[k];
  return l;
}

// W waves. ONE: all tokens are this block's and one sequence: no slots, the loss at once
template <int DT, int NE, int W, bool ONE>
__global__ __launch_bounds__(64 * W) void bal_fwd_kernel(BalArgs a) {
  typedef typename El<DT>::T T;
  __shared__ float sp[W][64 * NE];
  __shared__ int sc[MAX_E], sn;
  __shared__ float red[W];
  __shared__ long long tot[W];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, e0 = lane * NE;
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
      if (b >= e) continue;
    }
    for (int i = threadIdx.x; i < a.E; i += 64 * W) sc[i] = 0;
    if (threadIdx.x == 0) sn = 0;
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
    constexpr int B = TB<NE>;
    for (int64_t t0 = b + wave * B; t0 < e; t0 += W * B) {
      float z[B][NE];
      bool keep[B];
#pragma unroll
      for (int k = 0; k < B; ++k) {   // past the end: the last row again, with no share
        const int64_t t = min(t0 + k, e - 1);
        keep[k] = t0 + k < e;
        ld_run<DT, NE>((const T*)a.z + t * a.ldl, e0, a.E, -INFINITY, z[k]);
      }
      if (a.mask)
#pragma unroll
        for (int k = 0; k < B; ++k) {
          const bool counts = a.mask[min(t0 + k, e - 1)];
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
      over_wave<Max>(m);
#pragma unroll
      for (int k = 0; k < B; ++k) {
        sum[k] = 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) {   // experts past E are at -inf
          z[k][i] = exp_acc(z[k][i] - m[k]);
          sum[k] += z[k][i];
        }
      }
      over_wave<Sum>(sum);
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const float r = inverse(sum[k]), share = keep[k] ? r : 0.f;
#pragma unroll
        for (int i = 0; i < NE; ++i) acc[i] = fmaf(z[k][i], share, acc[i]);
        n += keep[k];
        if (a.rows && lane == 0 && t0 + k < e) a.rows[t0 + k] = Row{m[k], r, keep[k] ? s : -1, 0};
      }
    }
    while (i0 < e * a.K) {
      if (id >= 0 && id < a.E) atomicAdd(&sc[id], 1);
      i0 += 64 * W;
      id = pick(i0);
    }
    if (lane == 0) atomicAdd(&sn, n);
#pragma unroll
    for (int i = 0; i < NE; ++i) sp[wave][e0 + i] = acc[i];
    __syncthreads();
    auto share = [&](int x) {
      float P = sp[0][x];
#pragma unroll
      for (int k = 1; k < W; ++k) P += sp[k][x];
      return P;
    };
    if constexpr (ONE) {
      const int x = threadIdx.x;
      const float l = finish_seq(a, 0, x, x < a.E ? sc[x] : 0, sn, x < a.E ? share(x) : 0.f, red, tot);
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

// One sequence: its slots' sums, counts, weights and loss. Threads: columns of `1 << lgc` experts, the groups take every
// group-th slot each.
template <int BS>
__global__ __launch_bounds__(BS) void bal_seq_kernel(BalArgs a, int lgc) {
  __shared__ float sp[BS], red[BS / 64];
  __shared__ int sc[BS];
  __shared__ long long tot[BS / 64];
  __shared__ int sn;
  const int s = blockIdx.x;
  const int64_t b = a.q.at(s), e = a.q.at(s + 1);
  const int cols = 1 << lgc, groups = BS >> lgc, x = threadIdx.x & (cols - 1), g = threadIdx.x >> lgc;
  const int64_t k0 = b / a.chunk + s, k1 = b < e ? (e - 1) / a.chunk + s : k0 - 1;
  float P = 0.f;
  int c = 0;   // K T < 2^31
  if (x < a.E)
#pragma unroll 8
    for (int64_t k = k0 + g; k <= k1; k += groups) {
      P += a.P[k * a.E + x];
      c += a.C[k * a.E + x];
    }
  if (threadIdx.x < 64) {
    int n = 0;
    for (int64_t k = k0 + threadIdx.x; k <= k1; k += 64) n += a.N[k];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, 64);
    if (threadIdx.x == 0) sn = n;
  }
  sp[threadIdx.x] = P;
  sc[threadIdx.x] = c;
  __syncthreads();
  if (g == 0)
    for (int k = 1; k < groups; ++k) {
      P += sp[(k << lgc) + x];
      c += sc[(k << lgc) + x];
    }
  const int mine = g == 0 ? x : MAX_E;
  const float l = finish_seq(a, s, mine, c, sn, P, red, tot);
  if (threadIdx.x == 0) {
    if (a.q.S == 1) {
      *a.loss = l;
      a.weights[a.E] = 1.f;
    } else {
      a.seq_loss[s] = l;
      a.seq_n[s] = sn > 0;
    }
  }
}

__global__ __launch_bounds__(1024) void bal_join_kernel(BalArgs a) {
  __shared__ float red[16];
  __shared__ int cnt[16];
  float l = 0.f;
  int n = 0;
  for (int s = threadIdx.x; s < a.q.S; s += 1024) {
    l += a.seq_loss[s];
    n += a.seq_n[s];
  }
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

template <int DT, int NE>
__global__ __launch_bounds__(256) void bal_bwd_kernel(BalArgs a, const float* __restrict__ go, void* __restrict__ dz) {
  typedef typename El<DT>::T T;
  constexpr int B = TB<NE>;
  const int lane = threadIdx.x & 63, e0 = lane * NE;
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * B;
  if (t0 >= a.T) return;
  const float g = *go * a.weights[(int64_t)a.q.S * a.E];
  float z[B][NE], v[B][NE];
  Row row[B];
#pragma unroll
  for (int k = 0; k < B; ++k) {
    const int64_t t = min(t0 + k, a.T - 1);
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
  over_wave<Sum>(dot);
#pragma unroll
  for (int k = 0; k < B; ++k) {
    if (t0 + k >= a.T) break;
    float d[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) d[i] = row[k].seq >= 0 ? g * (z[k][i] * (v[k][i] - dot[k])) : 0.f;
    st_run<DT, NE>((T*)dz + (t0 + k) * a.E, e0, a.E, d);
  }
}

// ------------------------------------------------------------------------------------------------ host

// Sequences of under 64 tokens on average: blocks of four waves and about four sequences (each costs a block a few round
// trips to memory, so many blocks have to be under way: 131072 tokens in 4096 sequences 129 -> 40 us).
bool short_seqs(int64_t T, int64_t S) { return S > 1 && S * 64 > T; }
// tokens of a forward block: up to 256 blocks, 64 tokens at least (four for a wave)
int chunk_of(int64_t T, int64_t S) {
  if (short_seqs(T, S)) return (int)std::max<int64_t>(4, 4 * T / S);
  return (int)std::max<int64_t>((T + 255) / 256, 64);
}
int64_t chunks_of(int64_t T, int64_t S) { return T ? (T + chunk_of(T, S) - 1) / chunk_of(T, S) : 0; }
constexpr int64_t ONE_BLOCK = 192;   // tokens of one sequence that a block takes alone

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
  w.loss = w.N + up(slots * 4);
  w.n = w.loss + up(S * 4);
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
// f(dtype, experts a lane) as constants
template <class F>
void pick(int dtype, int64_t E, F f) {
  auto by_e = [&](auto dt) {
    if (E <= 64) f(dt, Int<1>{});
    else if (E <= 128) f(dt, Int<2>{});
    else if (E <= 256) f(dt, Int<4>{});
    else f(dt, Int<8>{});
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
    pick(dtype, E, [&](auto dt, auto ne) {
      bal_fwd_kernel<decltype(dt)::value, decltype(ne)::value, 16, true><<<1, 1024, 0, stream>>>(a);
    });
    return smel::launch_status();
  }
  a.chunk = chunk_of(T, S);
  a.P = (float*)(base + w.P);
  a.C = (int32_t*)(base + w.C);
  a.N = (int32_t*)(base + w.N);
  a.seq_loss = (float*)(base + w.loss);
  a.seq_n = (int32_t*)(base + w.n);
  if (T)
    pick(dtype, E, [&](auto dt, auto ne) {
      constexpr int d = decltype(dt)::value, m = decltype(ne)::value;
      const unsigned n = (unsigned)chunks_of(T, S);
      if (short_seqs(T, S)) bal_fwd_kernel<d, m, 4, false><<<n, 256, 0, stream>>>(a);
      else bal_fwd_kernel<d, m, 16, false><<<n, 1024, 0, stream>>>(a);
    });
  int lgc = 6;
  while ((1 << lgc) < E) ++lgc;
  if (S <= 512) bal_seq_kernel<1024><<<(unsigned)S, 1024, 0, stream>>>(a, lgc);
  else bal_seq_kernel<512><<<(unsigned)S, 512, 0, stream>>>(a, lgc);
  if (S > 1) bal_join_kernel<<<1, 1024, 0, stream>>>(a);
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
  pick(dtype, E, [&](auto dt, auto ne) {
    constexpr int tokens = 4 * TB<decltype(ne)::value>;
    bal_bwd_kernel<decltype(dt)::value, decltype(ne)::value><<<(unsigned)((T + tokens - 1) / tokens), 256, 0, stream>>>(a, go, dlogits);
  });
  return smel::launch_status();
}
