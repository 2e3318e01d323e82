// Balance loss of the router with its counts and gradient: for a sequence of n counted tokens with c_e picks of expert e,
//   L = E sum_e c_e / (K n) P_e,  P_e = mean_t p_te,  p_t = softmax(z_t)
//   dL/dz_te = p_te (v_e - sum_j p_tj v_j),  v_e = E c_e / (K n^2)      (the counts are constants)
// v only enters through differences, so its mean is taken out first: c_e - (sum c) / E is formed from whole numbers, and a
// balanced router's gradient is zero instead of the rounding of two equal terms.
//
// Forward: a block takes a chunk of tokens and walks through the sequences in it; per sequence, each wave's lanes sum the
// softmax of its rows per expert in registers (lane: experts l, l + 64, ...), the picks are counted by integer adds in LDS,
// and the block writes both to slot (chunk + sequence) of the workspace: along the tokens either number grows at every
// step, so slots are distinct and a sequence's are consecutive. A second kernel (a block per sequence) adds a sequence's
// slots in order; a third joins the sequences' losses where there are several. Sums have a fixed order, integer adds have
// none that shows: results repeat bit for bit. Backward: one pass, a row per wave.
#include "../../include/smel_loss.h"
#include "abi_util.h"
#include "common.h"

namespace {

constexpr int MAX_E = 512, MAX_K = 64;

template <int DT>
SMEL_DEV float ld_logit(const void* p, int64_t i) {
  if constexpr (DT == 1) return ((const float*)p)[i];
  const uint32_t b = ((const uint16_t*)p)[i];
  if constexpr (DT == 0) return __uint_as_float(b << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}

// e^x (x <= 0 or NaN) on v_exp_f32: x log2(e) in two parts, so that the product's rounding does not grow with |x|; an expert
// at -inf gives 0
SMEL_DEV float exp_acc(float x) {
  x = x < -200.f ? -200.f : x;
  const float hi = x * 1.4426950408889634f;
  const float lo = fmaf(x, 1.4426950408889634f, -hi) + x * 1.9259629911266175e-8f;
  return __builtin_amdgcn_exp2f(hi) * fmaf(lo, 0.6931471805599453f, 1.f);
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

struct BalArgs {
  const void* z;
  int64_t ldl, T;
  const void* topi;
  int topi_i64;
  int E, K, chunk, nchunk;
  const uint8_t* mask;
  Seqs q;
  float coef;
  float* row_stats;
  float* P;        // [slots][E]
  int32_t* C;      // [slots][E + 1]: picks, then counted tokens
  float* loss;
  int64_t* counts;
  float* weights;
  float* seq_loss; // [S]
  int32_t* seq_n;  // [S]
};

template <int DT, int NE>
__global__ __launch_bounds__(256) void bal_fwd_kernel(BalArgs a) {
  __shared__ float sp[4][MAX_E];
  __shared__ int sc[MAX_E + 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t c0 = (int64_t)blockIdx.x * a.chunk, c1 = min(c0 + a.chunk, a.T);
  int s = max(a.q.find(c0), 0);
  for (; s < a.q.S; ++s) {
    const int64_t b = max(a.q.at(s), c0), e = min(a.q.at(s + 1), c1);
    if (a.q.at(s) >= c1) break;
    if (b >= e) continue;
    for (int i = threadIdx.x; i <= a.E; i += 256) sc[i] = 0;
    __syncthreads();
    float acc[NE];
#pragma unroll
    for (int i = 0; i < NE; ++i) acc[i] = 0.f;
    for (int64_t t = b + wave; t < e; t += 4) {
      if (a.mask && !a.mask[t]) continue;
      float z[NE], m = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        const int x = lane + 64 * i;
        z[i] = x < a.E ? ld_logit<DT>(a.z, t * a.ldl + x) : -INFINITY;
        m = fmaxf(m, z[i]);
      }
      m = wave_max(m);
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        z[i] = lane + 64 * i < a.E ? exp_acc(z[i] - m) : 0.f;
        sum += z[i];
      }
      const float r = 1.f / wave_sum(sum);
#pragma unroll
      for (int i = 0; i < NE; ++i) acc[i] = fmaf(z[i], r, acc[i]);
      if (lane == 0) {
        if (a.row_stats) {
          a.row_stats[2 * t] = m;
          a.row_stats[2 * t + 1] = r;
        }
        atomicAdd(&sc[a.E], 1);
      }
    }
    for (int64_t i = b * a.K + threadIdx.x; i < e * a.K; i += 256) {
      if (a.mask && !a.mask[i / a.K]) continue;
      const int64_t id = a.topi_i64 ? ((const int64_t*)a.topi)[i] : (int64_t)((const int32_t*)a.topi)[i];
      if (id >= 0 && id < a.E) atomicAdd(&sc[id], 1);
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) sp[wave][lane + 64 * i] = acc[i];
    __syncthreads();
    const int64_t slot = (int64_t)blockIdx.x + s;
    for (int x = threadIdx.x; x <= a.E; x += 256) {
      if (x < a.E) a.P[slot * a.E + x] = ((sp[0][x] + sp[1][x]) + sp[2][x]) + sp[3][x];
      a.C[slot * (a.E + 1) + x] = sc[x];
    }
    __syncthreads();
  }
}

// one sequence: its slots' sums, counts, gradient weights and loss
__global__ __launch_bounds__(512) void bal_seq_kernel(BalArgs a) {
  __shared__ float red[8];
  __shared__ long long tot[8];
  const int s = blockIdx.x, x = threadIdx.x;   // an expert per thread
  const int64_t b = a.q.at(s), e = a.q.at(s + 1);
  int64_t c = 0;
  int64_t n = 0;
  float P = 0.f;
  if (b < e) {
    const int64_t k0 = b / a.chunk + s, k1 = (e - 1) / a.chunk + s;
    for (int64_t k = k0; k <= k1; ++k) {
      n += a.C[k * (a.E + 1) + a.E];
      if (x < a.E) {
        P += a.P[k * a.E + x];
        c += a.C[k * (a.E + 1) + x];
      }
    }
  }
  if (x < a.E) a.counts[(int64_t)s * a.E + x] = c;
  // picks in range, over all experts
  long long ct = c;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) ct += __shfl_xor(ct, o, 64);
  if ((x & 63) == 0) tot[x >> 6] = ct;
  __syncthreads();
  ct = 0;
  for (int k = 0; k < 8; ++k) ct += tot[k];
  float l = 0.f;
  if (x < a.E && n > 0) {
    const double scale = (double)a.coef / ((double)a.K * (double)n * (double)n);
    a.weights[(int64_t)s * a.E + x] = (float)((double)(c * a.E - ct) * scale);
    l = (float)((double)c * a.E * scale) * P;
  } else if (x < a.E) {
    a.weights[(int64_t)s * a.E + x] = 0.f;
  }
  l = wave_sum(l);
  if ((x & 63) == 0) red[x >> 6] = l;
  __syncthreads();
  if (x == 0) {
    for (int k = 1; k < 8; ++k) l += red[k];
    if (a.q.S == 1) {
      *a.loss = l;
      a.weights[a.E] = 1.f;
    } else {
      a.seq_loss[s] = l;
      a.seq_n[s] = n > 0;
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
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (t >= a.T) return;
  const int s = a.q.find(t);
  const bool counts = s >= 0 && s < a.q.S && t < a.q.at(s + 1) && !(a.mask && !a.mask[t]);
  float p[NE], d[NE];
  if (counts) {
    const float m = a.row_stats[2 * t], r = a.row_stats[2 * t + 1];
    const float g = *go * a.weights[(int64_t)a.q.S * a.E];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int x = lane + 64 * i;
      p[i] = x < a.E ? exp_acc(ld_logit<DT>(a.z, t * a.ldl + x) - m) * r : 0.f;
      d[i] = x < a.E ? a.weights[(int64_t)s * a.E + x] : 0.f;
      dot = fmaf(p[i], d[i], dot);
    }
    dot = wave_sum(dot);
#pragma unroll
    for (int i = 0; i < NE; ++i) d[i] = g * (p[i] * (d[i] - dot));
  } else {
#pragma unroll
    for (int i = 0; i < NE; ++i) d[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int x = lane + 64 * i;
    if (x >= a.E) continue;
    if constexpr (DT == 1) ((float*)dz)[t * a.E + x] = d[i];
    if constexpr (DT == 0) ((uint16_t*)dz)[t * a.E + x] = f2bf(d[i]);
    if constexpr (DT == 2) ((uint16_t*)dz)[t * a.E + x] = __builtin_bit_cast(uint16_t, (_Float16)d[i]);
  }
}

// ------------------------------------------------------------------------------------------------ host

int chunk_of(int64_t T) {
  int64_t c = (T + 255) / 256;
  return (int)(c < 16 ? 16 : c);
}
int64_t chunks_of(int64_t T) { return T ? (T + chunk_of(T) - 1) / chunk_of(T) : 0; }

struct Ws {
  int64_t P, C, loss, n, bytes;
};
Ws ws_of(int64_t T, int64_t E, int64_t S) {
  auto up = [](int64_t b) { return (b + 15) / 16 * 16; };
  const int64_t slots = chunks_of(T) + S;
  Ws w;
  w.P = 0;
  w.C = up(slots * E * 4);
  w.loss = w.C + up(slots * (E + 1) * 4);
  w.n = w.loss + up(S * 4);
  w.bytes = w.n + up(S * 4);
  return w;
}

int check(const char* name, const void* z, int64_t ldl, int dtype, int64_t T, int64_t E, int64_t S, const void* off) {
  SMEL_REQUIRE(T >= 0 && T <= (int64_t)1 << 25, SMEL_EUNSUPPORTED, "%s: T=%lld tokens, 0 to 2^25", name, (long long)T);
  SMEL_REQUIRE(E >= 1 && E <= MAX_E, SMEL_EUNSUPPORTED, "%s: E=%lld experts, 1 to %d", name, (long long)E, MAX_E);
  SMEL_REQUIRE(S >= 1 && S <= (int64_t)1 << 24, SMEL_EUNSUPPORTED, "%s: S=%lld sequences, 1 to 2^24", name, (long long)S);
  SMEL_REQUIRE(off || S == 1, SMEL_EINVAL, "%s: %lld sequences without offsets", name, (long long)S);
  SMEL_REQUIRE(dtype >= 0 && dtype <= 2, SMEL_EINVAL, "%s: dtype %d (0 = bf16, 1 = fp32, 2 = fp16)", name, dtype);
  SMEL_REQUIRE(T == 0 || z, SMEL_EINVAL, "%s: null logits", name);
  SMEL_REQUIRE(T <= 1 || ldl >= E, SMEL_EINVAL, "%s: row stride %lld < E=%lld", name, (long long)ldl, (long long)E);
  return 0;
}

// f<DT, NE> of the call's type and experts per lane
#define BAL_PICK(F, ...)                                                                        \
  [&](auto dt) {                                                                                \
    if (a.E <= 64) F<decltype(dt)::value, 1> __VA_ARGS__;                                       \
    else if (a.E <= 128) F<decltype(dt)::value, 2> __VA_ARGS__;                                 \
    else if (a.E <= 256) F<decltype(dt)::value, 4> __VA_ARGS__;                                 \
    else F<decltype(dt)::value, 8> __VA_ARGS__;                                                 \
  }
template <int V>
struct Int {
  static constexpr int value = V;
};
template <class F>
void by_dtype(int dtype, F f) {
  if (dtype == 0) f(Int<0>{});
  else if (dtype == 1) f(Int<1>{});
  else f(Int<2>{});
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
  char* const base = (char*)ws;
  BalArgs a{};
  a.z = logits;
  a.ldl = ldl;
  a.T = T;
  a.topi = topi;
  a.topi_i64 = topi_i64;
  a.E = (int)E;
  a.K = (int)K;
  a.chunk = chunk_of(T);
  a.nchunk = (int)chunks_of(T);
  a.mask = mask;
  a.q = Seqs{offsets, off_i64, (int)S, T};
  a.coef = coef;
  a.row_stats = row_stats;
  a.P = (float*)(base + w.P);
  a.C = (int32_t*)(base + w.C);
  a.loss = loss;
  a.counts = counts;
  a.weights = weights;
  a.seq_loss = (float*)(base + w.loss);
  a.seq_n = (int32_t*)(base + w.n);
  if (a.nchunk) by_dtype(dtype, BAL_PICK(bal_fwd_kernel, <<<a.nchunk, 256, 0, stream>>>(a)));
  bal_seq_kernel<<<(unsigned)S, 512, 0, stream>>>(a);
  if (S > 1) bal_join_kernel<<<1, 1024, 0, stream>>>(a);
  return smel::launch_status();
}

extern "C" int smel_balance_bwd(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E,
                                const uint8_t* mask, const void* offsets, int32_t off_i64, int64_t S,
                                const float* row_stats, const float* weights, const float* go, void* dlogits,
                                hipStream_t stream) {
  const int rc = check("balance_bwd", logits, ldl, dtype, T, E, S, offsets);
  if (rc) return rc;
  if (T == 0) return 0;
  SMEL_REQUIRE(row_stats && weights && go && dlogits, SMEL_EINVAL, "balance_bwd: null pointer");
  BalArgs a{};
  a.z = logits;
  a.ldl = ldl;
  a.T = T;
  a.E = (int)E;
  a.mask = mask;
  a.q = Seqs{offsets, off_i64, (int)S, T};
  a.row_stats = const_cast<float*>(row_stats);
  a.weights = const_cast<float*>(weights);
  by_dtype(dtype, BAL_PICK(bal_bwd_kernel, <<<(unsigned)((T + 3) / 4), 256, 0, stream>>>(a, go, dlogits)));
  return smel::launch_status();
}
