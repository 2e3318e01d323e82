// The choice of experts from router logits: sigmoid or softmax scores, a bias for the balance of the load, groups of experts, top-k,
// renormalised weights; and its backward.
//   s = sigmoid(z) | softmax(z);  c = s + bias;  the top_groups groups with the largest sum of their best one or two c stay;
//   ids = the K largest c, w_k = scale s_k / (sum_k s_k + 1e-20)
// One pass over the logits, and one for the gradient (sigmoid scores: the K picked logits alone). us: a token of 256 experts in eight
// groups 3.4; 4092 fp32 6.5 and 4.8; 32768 bf16 30 and 11 (bytes: 4 and 4); 131072 of 64 experts 24 and 15.
#include <math.h>

#include "abi_util.h"
#include "common.h"
#include "rows.h"

namespace {

constexpr int MAXE = 512;
constexpr int MAXK = 16;
constexpr int MAXG = 64;
constexpr float SUM_EPS = 1e-20f;

struct SelArgs {
  const void* z;
  const float* bias;
  float *topv, *scores, *stats;
  int64_t* topi;
  int64_t ldl, T;
  int E, K, score, best, renorm, drop;
  int parts, size, lg, per;   // groups, experts of one; log2 of a group's lanes; experts of a lane
  int top_groups;
  float scale;
};

template <int DT>
SMEL_DEV float logit_at(const void* z, int64_t at) {
  if constexpr (DT == 2)
    return ((const float*)z)[at];
  else
    return cvt<DT>(((const uint16_t*)z)[at]);
}
// 8 values kept in the caches for the next kernel (rows.h's stores pass them by)
template <int DT>
SMEL_DEV void keep8(typename El<DT>::T* p, int e0, int n, const Raw<DT>& r) {
  if constexpr (DT == 2) {
    store8<2, true>(p, e0, n, r);
  } else {
    if (e0 + 8 <= n) *(u32x4_a2*)(p + e0) = r.q[0];
    else store8<DT>(p, e0, n, r);
  }
}
// order-preserving form of a choice, above 0: -infinity and NaN are 0x007fffff
SMEL_DEV uint32_t order_of(float c) {
  if (!(c > -INFINITY)) return 0x007fffffu;
  const uint32_t b = __float_as_uint(c + 0.f);   // -0 is +0
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
SMEL_DEV float choice_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
// Reductions over the LT (16 or 64) lanes of a token, every lane gets the result. Within 16 lanes by DPP moves: a row's halves and
// quads are exchanged until all agree.
template <int CTRL>
SMEL_DEV uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
SMEL_DEV float dpp(float v) {
  return __uint_as_float(dpp<CTRL>(__float_as_uint(v)));
}
constexpr int XOR1 = 0xB1, XOR2 = 0x4E, HALF_MIRROR = 0x141, MIRROR = 0x140;
template <int LT, typename T, typename F>
SMEL_DEV T over_lanes(T v, F f, int from = 1) {   // from 2: pairs agree already
  if (from < 2) v = f(v, dpp<XOR1>(v));
  v = f(v, dpp<XOR2>(v));
  v = f(v, dpp<HALF_MIRROR>(v));
  v = f(v, dpp<MIRROR>(v));
  if (LT == 64) {
    v = f(v, __shfl_xor(v, 16, 64));
    v = f(v, __shfl_xor(v, 32, 64));
  }
  return v;
}
template <int LT>
SMEL_DEV float sum_lanes(float v) {
  return over_lanes<LT>(v, [](float a, float b) { return a + b; });
}
template <int LT>
SMEL_DEV uint32_t max_lanes(uint32_t v) {
  if constexpr (LT == 64) return wave_max_u32(v);
  return over_lanes<LT>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
// One score for the comparisons, the scores handed out, the weights and their gradients: the lower index of a tie and the weights'
// order are those of the numbers that a caller sees. Both are the rounded quotient in a few instructions (32768 tokens of 256 experts,
// events: 27.6 us, with divisions 28.0, with two scores, the compared ones from the bare reciprocal, 27.1).
// 1 / (1 + e^-z): one step of Newton's on the hardware's reciprocal is the quotient for every d below 2^126 (all 2^23 mantissas
// compared at seven exponents); 0 from there on, z < -87.3. An infinite d must not meet the reciprocal's 0; NaN stays NaN in r.
SMEL_DEV float sigmoid_of(float z) {
  const float d = 1.f + expf(-z), r = __builtin_amdgcn_rcpf(d);
  return fmaf(fmaf(-fminf(d, 0x1.fffffep127f), r, 1.f), r, r);
}
// e / den from den's rounded reciprocal (the quotient's bits from e = 2^-100 on); den: a softmax's sum, or for a row without a logit above -infinity (e = 0) one
SMEL_DEV float share_of(float e, float den, float inv) {
  const float q = e * inv;
  return fmaf(fmaf(-q, den, e), inv, q);
}
SMEL_DEV float den_of(float total) { return total == INFINITY ? 1.f : total; }

// n (<= N) values from p on, zeros behind; all of them at once where there are N
template <int DT, int N>
SMEL_DEV void run_of(const void* base, int64_t at, int n, float v[N]) {
  typedef typename El<DT>::T T;
  const T* const p = (const T*)base + at;
  if constexpr (N > 1) {
    if (n == N) {
      typedef T __attribute__((ext_vector_type(N < 8 ? N : 8), aligned(sizeof(T)))) vec;
#pragma unroll
      for (int i = 0; i < (N + 7) / 8; ++i) {
        const vec q = ((const vec*)p)[i];
#pragma unroll
        for (int j = 0; j < (N < 8 ? N : 8); ++j) {
          if constexpr (DT == 2) v[8 * i + j] = q[j];
          else v[8 * i + j] = cvt<DT>((uint32_t)q[j]);
        }
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = j < n ? logit_at<DT>(p, j) : 0.f;
}

// The sum of a softmax's terms (n of a lane's N): neighbours in pairs, pairs of pairs, ...; from 128 experts on fours are added up one
// after the other first. For powers of two up to 256 that is one order, however many lanes a token has: with one pick and
// renormalised weights the gradient is nothing but the roundings of d s / s, and those do not change with the batch.
template <int LT, int N>
SMEL_DEV float row_total(const float (&s)[N], int n, int E) {
  float v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = j < n ? s[j] : 0.f;
  if constexpr (N == 1) return sum_lanes<LT>(v[0]);
  if constexpr (N == 2) {
    float a = v[0] + v[1];
    if (E >= 128) {   // the even lane of two goes on with the other's
      const float c = dpp<XOR1>(v[0]), d = dpp<XOR1>(v[1]);
      a = lane_id() & 1 ? (c + d + v[0]) + v[1] : (a + c) + d;
      a = over_lanes<LT>(a, [](float p, float q) { return p + q; }, 2);
      return a;
    }
    return sum_lanes<LT>(a);
  }
  float q[N / 4 > 0 ? N / 4 : 1];
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    q[i] = E >= 128 ? ((v[4 * i] + v[4 * i + 1]) + v[4 * i + 2]) + v[4 * i + 3] : (v[4 * i] + v[4 * i + 1]) + (v[4 * i + 2] + v[4 * i + 3]);
#pragma unroll
  for (int o = 1; o < N / 4; o *= 2)
#pragma unroll
    for (int i = 0; i + o < N / 4; i += 2 * o) q[i] += q[i + o];
  return sum_lanes<LT>(q[0]);
}

template <int N>
struct Order {
  typedef uint32_t T;
};
template <>
struct Order<16> {
  typedef uint64_t T;
};

// LT lanes a token (four tokens a wave, or one). A group's experts lie in LT / 2^k lanes next to each other, N of them at most in a
// lane, in the order of their indices; without groups to drop, all experts are one. Each lane sorts its own, so a pick is the largest
// of the lanes' heads: the maximum by DPP moves, the lowest lane that holds it (the lowest index: ties), and that lane goes on to its
// next. Bound by instructions: about 22 for a pick, 18 for a score, 5 for each of a lane's N (N - 1) / 2 comparisons.
template <int DT, int LT, int N>
__global__ __launch_bounds__(256) void select_kernel(SelArgs p) {
  const int l = lane_id(), li = l & (LT - 1), base = l & ~(LT - 1);
  const int64_t t = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / LT) + l / LT;
  const bool live = t < p.T;
  const int64_t row = live ? t : p.T - 1;
  const int grp = li >> p.lg, q = li & ((1 << p.lg) - 1);
  const int e0 = grp * p.size + q * p.per;
  const int n = grp < p.parts ? min(max(p.size - q * p.per, 0), p.per) : 0;
  float s[N], bias[N];
  run_of<DT, N>(p.z, row * p.ldl + e0, n, s);
  if (p.bias) run_of<2, N>(p.bias, e0, n, bias);
  float m = 0.f, den = 1.f, inv = 1.f;
  if (p.score == 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = sigmoid_of(s[j]);
  } else {
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) m = fmaxf(m, s[j]);
    m = over_lanes<LT>(m, [](float a, float b) { return fmaxf(a, b); });
    if (!(m > -INFINITY)) m = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = expf(s[j] - m);
    float sum = row_total<LT, N>(s, n, p.E);
    if (sum == 0.f) sum = INFINITY;     // no logit above -infinity: scores 0
    den = den_of(sum);
    inv = 1.f / den;
#pragma unroll
    for (int j = 0; j < N; ++j) s[j] = share_of(s[j], den, inv);
    if (p.stats && live && li == 0) {
      p.stats[2 * t] = m;
      p.stats[2 * t + 1] = sum;
    }
  }
  if (p.scores && live)
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) p.scores[t * p.E + e0 + j] = s[j];
  uint32_t key[N], at[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    key[j] = j < n ? order_of(p.bias ? s[j] + bias[j] : s[j]) : 0u;
    at[j] = j;
  }
  // descending, equal ones in order
#pragma unroll
  for (int i = 1; i < N; ++i)
#pragma unroll
    for (int j = N - 1; j >= i; --j) {
      const uint32_t k1 = key[j], k0 = key[j - 1], a1 = at[j], a0 = at[j - 1];
      const bool up = k1 > k0;
      key[j - 1] = max(k1, k0);
      key[j] = min(k1, k0);
      at[j - 1] = up ? +a1 : +a0;   // of values: a conditional of the variables themselves is one of addresses
      at[j] = up ? +a0 : +a1;
    }
  if (p.drop) {   // groups
    float c1 = key[0] ? choice_of(key[0]) : -INFINITY, c2 = -INFINITY;
    if constexpr (N > 1) c2 = key[1] ? choice_of(key[1]) : -INFINITY;
    auto join = [&](float d1, float d2) {
      c2 = fmaxf(fminf(c1, d1), fmaxf(c2, d2));
      c1 = fmaxf(c1, d1);
    };
    if (p.lg > 0) join(dpp<XOR1>(c1), dpp<XOR1>(c2));
    if (p.lg > 1) join(dpp<XOR2>(c1), dpp<XOR2>(c2));
    if (p.lg > 2) join(dpp<HALF_MIRROR>(c1), dpp<HALF_MIRROR>(c2));
    if (p.lg > 3) join(dpp<MIRROR>(c1), dpp<MIRROR>(c2));
    if (p.lg > 4) join(__shfl_xor(c1, 16, 64), __shfl_xor(c2, 16, 64));
    const uint32_t value = grp < p.parts ? order_of(p.best == 2 && p.size > 1 ? c1 + c2 : c1) : 0u;
    int rank = 0;
    for (int g = 0; g < p.parts; ++g) {
      uint32_t v;
      if constexpr (LT == 64) v = (uint32_t)lane_get((int)value, g << p.lg);
      else v = __shfl(value, base + (g << p.lg), 64);
      rank += v > value || (v == value && g < grp);
    }
    if (rank >= p.top_groups)
#pragma unroll
      for (int j = 0; j < N; ++j) key[j] = 0u;
  }
  // the order of a lane's experts, four bits each
  typename Order<N>::T next = 0;
#pragma unroll
  for (int j = N - 1; j >= 0; --j) next = next << 4 | at[j];
  int id = 0;   // lane k of a token keeps pick k
  for (int k = 0; k < p.K; ++k) {
    const uint32_t best = max_lanes<LT>(key[0]);
    const uint64_t who = __ballot(key[0] == best);
    const int head = e0 + (int)(next & 15);
    int w;
    if constexpr (LT == 64) {
      w = __builtin_ctzll(who);
      const int e = lane_get(head, w);
      if (li == k) id = e;
    } else {
      w = __builtin_ctz((uint32_t)(who >> base) & 0xffffu);
      const int e = __shfl(head, base + w, 64);
      if (li == k) id = e;
    }
    if (li == w) {
#pragma unroll
      for (int j = 0; j + 1 < N; ++j) key[j] = key[j + 1];
      key[N - 1] = 0u;
      next >>= 4;
    }
  }
  float w = 0.f;
  if (li < p.K) {
    const float z = logit_at<DT>(p.z, row * p.ldl + id);
    w = p.score == 0 ? sigmoid_of(z) : share_of(expf(z - m), den, inv);
  }
  const float sum = sum_lanes<16>(w);   // K <= 16
  if (live && li < p.K) {
    p.topv[t * p.K + li] = p.renorm ? p.scale * w / (sum + SUM_EPS) : p.scale * w;
    p.topi[t * p.K + li] = id;
  }
}

// Order of a wave's LDS accesses for its lanes that exchange values there: the hardware keeps it, the compiler must too
SMEL_DEV void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct SelBwdArgs {
  const void* z;
  const int64_t* topi;
  const float *dtopv, *stats;
  void* dz;
  int64_t ldl, ldd, T;
  int E, K, score, renorm, lpr;
  float scale;
};

// lpr lanes a token, 8 columns each: lane k works out pick k's gradient and puts it into the row in LDS, each lane writes its columns.
// A row's lanes are of one wave. 32768 x 256 bf16 sigmoid 11 us, 131072 x 64 softmax 15: the bytes of dz (softmax: and of z) are 4 and 8.
// What is above them is a token's chain, with no second token on its way: the pick, its logit, the sums, LDS, the store.
template <int DT>
__global__ __launch_bounds__(256) void select_bwd_kernel(SelBwdArgs p) {
  typedef typename El<DT>::T T;
  __shared__ __attribute__((aligned(16))) float rows[256 * 8];
  const int lpr = p.lpr, li = threadIdx.x & (lpr - 1);
  const int64_t t = (int64_t)blockIdx.x * (256 / lpr) + threadIdx.x / lpr;
  const bool live = t < p.T;
  const int64_t row = live ? t : p.T - 1;
  float* const mine = rows + (threadIdx.x / lpr) * (8 * lpr);
  Raw<DT> z{};
  if (p.score && 8 * li < p.E) z = load8<DT>((const T*)p.z + row * p.ldl, 8 * li, p.E);
  f32x4_t* const own = (f32x4_t*)(mine + 8 * li);
  own[0] = own[1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  wave_lds_order();
  const float m = p.score ? p.stats[2 * row] : 0.f, total = p.score ? p.stats[2 * row + 1] : 1.f;
  int id = -1;
  float d = 0.f, s = 0.f, slope = 1.f;   // lane k: pick k
  if (li < p.K) {
    const int64_t e = p.topi[row * p.K + li];
    if (e >= 0 && e < p.E) {
      id = (int)e;
      d = p.scale * p.dtopv[row * p.K + li];
      const float zk = logit_at<DT>(p.z, row * p.ldl + id);
      if (p.score == 0) {
        s = sigmoid_of(zk);
        const float q = expf(-fabsf(zk)), a = __builtin_amdgcn_rcpf(1.f + q);
        slope = q * a * a;
      } else {
        const float den = den_of(total);
        s = share_of(expf(zk - m), den, 1.f / den);
      }
    }
  }
  auto sum = [&](float v) {
    for (int o = 1; o < lpr; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
  };
  if (p.renorm) {   // K = 1: the weight is a constant, and the difference what is left of d s / s
    const float S = sum(s) + SUM_EPS, dot = sum(d * s);
    d = (d - dot / S) / S;
  }
  const float all = p.score ? sum(d * s) : 0.f;
  if (id >= 0) atomicAdd(&mine[id], d * slope);
  wave_lds_order();
  if (!live) return;
  const f32x4_t a = own[0], b = own[1];
  float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  if (p.score) {
    const float inv = 1.f / total;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 8 * li + j < p.E ? expf(z.at(j) - m) * inv * (v[j] - all) : 0.f;
  }
  Raw<DT> o;
  o.set(v);
  T* const out = (T*)p.dz + t * p.ldd;
  const int n = (int)(p.ldd < 8 * lpr ? p.ldd : 8 * lpr);
  if (8 * li < n) keep8<DT>(out, 8 * li, n, o);
  for (int64_t e = 8 * lpr + li; e < p.ldd; e += lpr) out[e] = T(0);
}

// A lane's experts with lt lanes a token: their most, and log2 of the lanes of a group
int lane_plan(SelArgs& p, int lt) {
  int lanes = lt;
  p.lg = lt == 64 ? 6 : 4;
  for (int g = 1; g < p.parts; g *= 2) {
    lanes /= 2;
    --p.lg;
  }
  if (lanes == 0) return 1 << 20;
  return p.per = (p.size + lanes - 1) / lanes;
}
template <int DT, int LT, int N>
int launch_plan(const SelArgs& p, hipStream_t stream) {
  constexpr int64_t TOKENS = 4 * (64 / LT);
  select_kernel<DT, LT, N><<<(unsigned)((p.T + TOKENS - 1) / TOKENS), 256, 0, stream>>>(p);
  return smel::launch_status();
}
template <int DT>
int launch_select(SelArgs& p, hipStream_t stream) {
  // Four tokens a wave share a pick's instructions, but wait for each other and sort longer lists. us of the kernel, a token a wave and
  // four: 64 experts 4092 tokens 3.4, 3.3, 65536 tokens 21, 12; 128 experts 517 tokens 3.0, 3.9, 4092 4.1, 4.1, 65536 32, 21; lists of
  // 16 (256 experts) 65536 tokens 43, 78
  if (p.T >= 4096) {
    const int m = lane_plan(p, 16);
    if (m <= 4) return launch_plan<DT, 16, 4>(p, stream);
    if (m <= 8) return launch_plan<DT, 16, 8>(p, stream);
  }
  const int n = lane_plan(p, 64);
  if (n <= 1) return launch_plan<DT, 64, 1>(p, stream);
  if (n <= 2) return launch_plan<DT, 64, 2>(p, stream);
  if (n <= 4) return launch_plan<DT, 64, 4>(p, stream);
  if (n <= 8) return launch_plan<DT, 64, 8>(p, stream);
  // 256 registers, one wave a SIMD: 32768 tokens of 510 experts in 17 groups 232 us, of 512 in 16 46. Reached by 3 groups of more than 128
  // experts, 5 to 7 of more than 64, 9 to 15 of more than 32, 17 to 30 of more than 16, 33 and more of more than 8
  return launch_plan<DT, 64, 16>(p, stream);
}

int check(const char* name, int64_t ldl, int32_t dtype, int64_t T, int64_t E, int64_t K, int32_t score) {
  SMEL_REQUIRE(T >= 0 && E > 0 && K > 0, SMEL_EINVAL, "%s: bad sizes", name);
  SMEL_REQUIRE(T <= (int64_t)1 << 25, SMEL_EUNSUPPORTED, "%s: %lld tokens, at most 2^25", name, (long long)T);
  SMEL_REQUIRE(E <= MAXE, SMEL_EUNSUPPORTED, "%s: %lld experts, at most %d", name, (long long)E, MAXE);
  SMEL_REQUIRE(K <= E && K <= MAXK, SMEL_EUNSUPPORTED, "%s: top_k=%lld must be <= min(E, %d)", name, (long long)K, MAXK);
  SMEL_REQUIRE(dtype >= 0 && dtype <= 2, SMEL_EINVAL, "%s: dtype %d (0 = bf16, 1 = fp16, 2 = fp32)", name, dtype);
  SMEL_REQUIRE(score == 0 || score == 1, SMEL_EINVAL, "%s: score %d (0 = sigmoid, 1 = softmax)", name, score);
  SMEL_REQUIRE(T <= 1 || ldl >= E, SMEL_EINVAL, "%s: row stride %lld < %lld experts", name, (long long)ldl, (long long)E);
  return 0;
}

}  // namespace

extern "C" int smel_select_experts(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E, int64_t K, int32_t score,
                                   const float* bias, int64_t groups, int64_t top_groups, int32_t group_best, int32_t renorm,
                                   float scale, float* topv, int64_t* topi, float* scores, float* stats, hipStream_t stream) {
  const int rc = check("select_experts", ldl, dtype, T, E, K, score);
  if (rc) return rc;
  SMEL_REQUIRE(groups >= 1 && groups <= MAXG && E % groups == 0, SMEL_EUNSUPPORTED,
               "select_experts: %lld groups of %lld experts (1 to %d, of equal size)", (long long)groups, (long long)E, MAXG);
  SMEL_REQUIRE(top_groups >= 1 && top_groups <= groups && K <= top_groups * (E / groups), SMEL_EINVAL,
               "select_experts: %lld groups kept of %lld hold fewer than %lld experts", (long long)top_groups, (long long)groups,
               (long long)K);
  SMEL_REQUIRE(group_best == 1 || group_best == 2, SMEL_EINVAL, "select_experts: group_best %d (1 or 2)", group_best);
  if (T == 0) return 0;
  SMEL_REQUIRE(logits && topv && topi, SMEL_EINVAL, "select_experts: null pointer");
  SelArgs p{};
  p.z = logits;
  p.bias = bias;
  p.topv = topv;
  p.scores = scores;
  p.stats = stats;
  p.topi = topi;
  p.ldl = ldl;
  p.T = T;
  p.E = (int)E;
  p.K = (int)K;
  p.score = score;
  p.best = group_best;
  p.renorm = renorm;
  p.drop = top_groups < groups;
  p.parts = p.drop ? (int)groups : 1;
  p.size = p.E / p.parts;
  p.top_groups = (int)top_groups;
  p.scale = scale;
  return dtype == 0 ? launch_select<0>(p, stream) : dtype == 1 ? launch_select<1>(p, stream) : launch_select<2>(p, stream);
}

extern "C" int smel_select_experts_bwd(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E, int64_t K,
                                       int32_t score, int32_t renorm, float scale, const int64_t* topi, const float* dtopv,
                                       const float* stats, void* dlogits, int64_t ldd, hipStream_t stream) {
  const int rc = check("select_experts_bwd", ldl, dtype, T, E, K, score);
  if (rc) return rc;
  SMEL_REQUIRE(ldd >= E && ldd < (1 << 20), SMEL_EINVAL, "select_experts_bwd: row stride %lld for %lld experts", (long long)ldd, (long long)E);
  if (T == 0) return 0;
  SMEL_REQUIRE(logits && topi && dtopv && dlogits && (score == 0 || stats), SMEL_EINVAL, "select_experts_bwd: null pointer");
  int lpr = 1;
  while (lpr < 64 && (8 * lpr < E || lpr < K)) lpr *= 2;   // 8 lpr >= E, lpr >= K
  const SelBwdArgs p{logits, topi, dtopv, stats, dlogits, ldl, ldd, T, (int)E, (int)K, score, renorm, lpr, scale};
  const int64_t tokens = 256 / lpr;
  const dim3 g((unsigned)((T + tokens - 1) / tokens)), b(256);
  if (dtype == 0) select_bwd_kernel<0><<<g, b, 0, stream>>>(p);
  else if (dtype == 1) select_bwd_kernel<1><<<g, b, 0, stream>>>(p);
  else select_bwd_kernel<2><<<g, b, 0, stream>>>(p);
  return smel::launch_status();
}
