// gfx950 kernels of log probabilities of tokens, entropy and alternatives, and of their gradient.
//
//   lse = m + log s,  s = sum e^(x-m),  log_prob = x_target - lse,  entropy = log s - w / s,  w = sum (x-m) e^(x-m)
//   D_v = d_log_prob (1[v = target] - p_v) - d_entropy p_v (log p_v + entropy)
#pragma once

#include "sequence_common.h"

namespace rtn {

constexpr int kMaxAlternatives = 64;

struct ScoresArgs {
  const void* logits;
  long long ld;
  const int64_t* targets;
  long long rows, V;
  int top_k;
  float *log_prob, *norm, *entropy, *top_log_prob;
  int64_t* top_ids;
  const float *d_log_prob, *d_entropy;
  void* D;
};

// A logit and its index as one number that orders alternatives: larger is better.  A NaN comes before everything, -0 and 0 are equal,
// among equal logits the lower index is better.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);  // (-0 + 0 is 0)
  return x != x ? 0xFFFFFFFFu : (u & 0x80000000u ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long alternative(float x, unsigned index) { return (unsigned long long)order_of(x) << 32 | (unsigned)~index; }
__device__ __forceinline__ float logit_of(unsigned long long a) {
  const unsigned u = (unsigned)(a >> 32);
  return __builtin_bit_cast(float, u == 0xFFFFFFFFu ? 0x7FC00000u : (u & 0x80000000u ? u & 0x7FFFFFFFu : ~u));
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* shared, F join) {
  __syncthreads();
  shared[threadIdx.x] = v;
  __syncthreads();
  for (int half = blockDim.x / 2; half > 0; half /= 2) {
    if ((int)threadIdx.x < half) shared[threadIdx.x] = join(shared[threadIdx.x], shared[threadIdx.x + half]);
    __syncthreads();
  }
  return shared[0];
}

// One workgroup per row: the maximum, the sums, then the alternatives one by one.
template <typename AT>
__global__ __launch_bounds__(256) void k_token_scores(ScoresArgs a) {
  __shared__ float shared[256];
  __shared__ unsigned long long best_of[256];
  const long long r = blockIdx.x;
  const AT* x = (const AT*)a.logits + r * a.ld;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    if (threadIdx.x == 0) {
      if (a.log_prob) a.log_prob[r] = 0.f;
      if (a.norm) a.norm[2 * r] = a.norm[2 * r + 1] = 0.f;
      if (a.entropy) a.entropy[r] = 0.f;
    }
    for (int k = threadIdx.x; k < a.top_k; k += blockDim.x) {
      a.top_log_prob[r * a.top_k + k] = -__builtin_inff();
      a.top_ids[r * a.top_k + k] = -1;
    }
    return;
  }
  const float inf = __builtin_inff();
  float m = -inf, s = 0.f, w = 0.f;
  for (long long v = threadIdx.x; v < a.V; v += blockDim.x) {
    const float l = load_f32(x + v);
    m = l > m || l != l ? l : m;
  }
  m = block_reduce(m, shared, [](float p, float q) { return p != p || p > q ? p : q; });
  const float base = m == -inf ? 0.f : m;
  for (long long v = threadIdx.x; v < a.V; v += blockDim.x) {
    const float d = load_f32(x + v) - base, e = __expf(d);
    s += e;
    w += (d < -1e4f ? -1e4f : d) * e;  // (a NaN stays)
  }
  s = block_reduce(s, shared, [](float p, float q) { return p + q; });
  w = block_reduce(w, shared, [](float p, float q) { return p + q; });
  const float log_s = logf(s);
  auto log_prob_of = [&](float l) { return l == -inf ? -inf : (l - base) - log_s; };
  if (threadIdx.x == 0) {
    if (a.norm) a.norm[2 * r] = base, a.norm[2 * r + 1] = log_s;
    if (a.log_prob) a.log_prob[r] = target < a.V ? log_prob_of(load_f32(x + target)) : __builtin_nanf("");
    if (a.entropy) a.entropy[r] = m == -inf ? 0.f : log_s - w / s;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long best = 0;
    for (long long v = threadIdx.x; v < a.V; v += blockDim.x) {
      const unsigned long long q = alternative(load_f32(x + v), (unsigned)v);
      if (q > best && (k == 0 || q < last)) best = q;
    }
    best = block_reduce(best, best_of, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
    if (threadIdx.x == 0) {
      a.top_log_prob[r * a.top_k + k] = log_prob_of(logit_of(best));
      a.top_ids[r * a.top_k + k] = (int64_t)(unsigned)~(unsigned)best;
    }
    last = best;
  }
}

template <typename AT>
__global__ __launch_bounds__(256) void k_token_scores_bwd(ScoresArgs a) {
  const long long r = blockIdx.x;
  const AT* x = (const AT*)a.logits + r * a.ld;
  AT* D = (AT*)a.D + r * a.V;
  const long long target = a.targets ? a.targets[r] : 0;
  const float base = a.norm[2 * r], log_s = a.norm[2 * r + 1];
  const float g = a.d_log_prob && a.targets ? a.d_log_prob[r] : 0.f, ge = a.d_entropy ? a.d_entropy[r] : 0.f, h = a.d_entropy ? a.entropy[r] : 0.f;
  const bool none = target < 0 || log_s == -__builtin_inff(), bad = a.targets && target >= a.V;
  for (long long v = threadIdx.x; v < a.V; v += blockDim.x) {
    float d = 0.f;
    if (bad) {
      d = __builtin_nanf("");
    } else if (!none) {
      const float log_p = (load_f32(x + v) - base) - log_s, p = __expf(log_p);
      d = -p * (g + ge * ((log_p < -1e4f ? -1e4f : log_p) + h));
      if (a.targets && v == target) d += g;
    }
    store_f32(D + v, d);
  }
}

}  // namespace rtn
