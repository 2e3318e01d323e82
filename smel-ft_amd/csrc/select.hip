// The choice of experts from router logits: sigmoid or softmax scores, a bias for the balance of the load, groups of experts, top-k,
// renormalised weights; and its backward.
//   s = sigmoid(z) | softmax(z);  c = s + bias;  the top_groups groups with the largest sum of their best one or two c stay;
//   ids = the K largest c, w_k = scale s_k / (sum_k s_k + 1e-20)
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
  int E, K, score, groups, top_groups, best, renorm;
  float scale;
};

template <int DT>
SMEL_DEV float logit_at(const void* z, int64_t at) {
  if constexpr (DT == 2)
    return ((const float*)z)[at];
  else
    return cvt<DT>(((const uint16_t*)z)[at]);
}
// order-preserving form of a choice, above 0: -infinity and NaN are 0x007fffff
SMEL_DEV uint32_t order_of(float c) {
  if (!(c > -INFINITY)) return 0x007fffffu;
  const uint32_t b = __float_as_uint(c + 0.f);   // -0 is +0
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
SMEL_DEV float choice_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
SMEL_DEV uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t u = __shfl_xor(v, o, 64);
    v = v > u ? v : u;
  }
  return v;
}
SMEL_DEV float sigmoid_of(float z) { return 1.f / (1.f + expf(-z)); }

// a wave per token, expert l + 64 j in lane l
template <int DT>
__global__ __launch_bounds__(256) void select_kernel(SelArgs p) {
  constexpr int NPL = MAXE / 64;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const int l = lane_id();
  float s[NPL];
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int e = l + 64 * j;
    s[j] = e < p.E ? logit_at<DT>(p.z, t * p.ldl + e) : -INFINITY;
    m = fmaxf(m, s[j]);
  }
  if (p.score == 0) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] = sigmoid_of(s[j]);
  } else {
    m = wave_max(m);
    const float base = m > -INFINITY ? m : 0.f;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      s[j] = l + 64 * j < p.E ? expf(s[j] - base) : 0.f;
      sum += s[j];
    }
    sum = wave_sum(sum);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NPL; ++j) s[j] *= inv;
    if (p.stats && l == 0) {
      p.stats[2 * t] = base;
      p.stats[2 * t + 1] = inv;
    }
  }
  uint64_t key[NPL];
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int e = l + 64 * j;
    key[j] = 0;
    if (e < p.E) {
      if (p.scores) p.scores[t * p.E + e] = s[j];
      key[j] = (uint64_t)order_of(p.bias ? s[j] + p.bias[e] : s[j]) << 32 | (0xffffffffu - (uint32_t)e);
    }
  }
  const int size = p.E / p.groups;
  if (p.top_groups < p.groups) {
    uint64_t mine = 0;   // lane g keeps group g's value
    for (int g = 0; g < p.groups; ++g) {
      uint64_t first = 0, second = 0;
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if ((l + 64 * j) / size == g && key[j] > first) first = key[j];
      first = wave_max_u64(first);
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if ((l + 64 * j) / size == g && key[j] != first && key[j] > second) second = key[j];
      second = wave_max_u64(second);
      float v = choice_of(first >> 32);
      if (p.best == 2 && size > 1) v += choice_of(second >> 32);
      if (l == g) mine = (uint64_t)order_of(v) << 32 | (0xffffffffu - (uint32_t)g);
    }
    uint64_t kept = 0;
    for (int k = 0; k < p.top_groups; ++k) {
      const uint64_t b = wave_max_u64(mine);
      const int g = (int)(0xffffffffu - (uint32_t)b);
      kept |= 1ull << g;
      if (l == g) mine = 0;
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (l + 64 * j < p.E && !(kept >> ((l + 64 * j) / size) & 1)) key[j] = 0;
  }
  float w = 0.f, sum = 0.f;   // lane k keeps pick k
  int id = 0;
  for (int k = 0; k < p.K; ++k) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) best = best > key[j] ? best : key[j];
    best = wave_max_u64(best);
    const int e = (int)(0xffffffffu - (uint32_t)best);
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (l + 64 * j == e) {
        v = s[j];
        key[j] = 0;
      }
    v = __shfl(v, e & 63, 64);
    sum += v;
    if (l == k) {
      w = v;
      id = e;
    }
  }
  if (l < p.K) {
    p.topv[t * p.K + l] = p.renorm ? p.scale * w / (sum + SUM_EPS) : p.scale * w;
    p.topi[t * p.K + l] = id;
  }
}

struct SelBwdArgs {
  const void* z;
  const int64_t* topi;
  const float *dtopv, *stats;
  void* dz;
  int64_t ldl, ldd, T;
  int E, K, score, renorm;
  float scale;
};

template <int DT>
__global__ __launch_bounds__(256) void select_bwd_kernel(SelBwdArgs p) {
  typedef typename El<DT>::T T;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.T) return;
  const int l = lane_id();
  const float m = p.score ? p.stats[2 * t] : 0.f, inv = p.score ? p.stats[2 * t + 1] : 0.f;
  int id = -1;
  float d = 0.f, s = 0.f, slope = 0.f;   // lane k: pick k
  if (l < p.K) {
    const int64_t e = p.topi[t * p.K + l];
    if (e >= 0 && e < p.E) {
      id = (int)e;
      d = p.scale * p.dtopv[t * p.K + l];
      const float z = logit_at<DT>(p.z, t * p.ldl + id);
      if (p.score == 0) {
        s = sigmoid_of(z);
        const float q = expf(-fabsf(z));
        slope = q / ((1.f + q) * (1.f + q));
      } else {
        s = expf(z - m) * inv;
      }
    }
  }
  if (p.renorm) {
    const float S = wave_sum(s) + SUM_EPS, dot = wave_sum(d * s);
    d = (d - dot / S) / S;
  }
  const float all = p.score ? wave_sum(d * s) : 0.f;
  if (p.score == 0) d *= slope;
  for (int e = l; e < p.ldd; e += 64) {
    float g = 0.f;
    for (int k = 0; k < p.K; ++k) {
      const int ik = lane_get(id, k);
      const float dk = lane_get(d, k);
      if (ik == e) g += dk;
    }
    float v = g;
    if (p.score) v = e < p.E ? expf(logit_at<DT>(p.z, t * p.ldl + e) - m) * inv * (g - all) : 0.f;
    if constexpr (DT == 2)
      ((T*)p.dz)[t * p.ldd + e] = v;
    else
      ((T*)p.dz)[t * p.ldd + e] = (T)enc<DT>(v);
  }
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
  const SelArgs p{logits, bias,       topv,     scores,     stats,           topi,       ldl,    T,
                  (int)E, (int)K, score, (int)groups, (int)top_groups, group_best, renorm, scale};
  const dim3 g((unsigned)((T + 3) / 4)), b(256);
  if (dtype == 0) select_kernel<0><<<g, b, 0, stream>>>(p);
  else if (dtype == 1) select_kernel<1><<<g, b, 0, stream>>>(p);
  else select_kernel<2><<<g, b, 0, stream>>>(p);
  return smel::launch_status();
}

extern "C" int smel_select_experts_bwd(const void* logits, int64_t ldl, int32_t dtype, int64_t T, int64_t E, int64_t K,
                                       int32_t score, int32_t renorm, float scale, const int64_t* topi, const float* dtopv,
                                       const float* stats, void* dlogits, int64_t ldd, hipStream_t stream) {
  const int rc = check("select_experts_bwd", ldl, dtype, T, E, K, score);
  if (rc) return rc;
  SMEL_REQUIRE(ldd >= E && ldd < (1 << 20), SMEL_EINVAL, "select_experts_bwd: row stride %lld for %lld experts", (long long)ldd, (long long)E);
  if (T == 0) return 0;
  SMEL_REQUIRE(logits && topi && dtopv && dlogits && (score == 0 || stats), SMEL_EINVAL, "select_experts_bwd: null pointer");
  const SelBwdArgs p{logits, topi, dtopv, stats, dlogits, ldl, ldd, T, (int)E, (int)K, score, renorm, scale};
  const dim3 g((unsigned)((T + 3) / 4)), b(256);
  if (dtype == 0) select_bwd_kernel<0><<<g, b, 0, stream>>>(p);
  else if (dtype == 1) select_bwd_kernel<1><<<g, b, 0, stream>>>(p);
  else select_bwd_kernel<2><<<g, b, 0, stream>>>(p);
  return smel::launch_status();
}
