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
  int splits;          // pieces of a row
  long long segment;   // logits of a piece
  float* part;         // [rows][splits][4] of the pieces: maximum, sums
  unsigned long long* part_top;  // [rows][splits][top_k]
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

// ---- over the 64 lanes of a wavefront, the same result in all of them ----
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
template <typename F>
__device__ __forceinline__ float over_wave(float v, F join) {
  v = join(v, dpp<0xB1>(v));   // the neighbour of a pair
  v = join(v, dpp<0x4E>(v));   // the other pair of four
  v = join(v, dpp<0x141>(v));  // the other half of eight, mirrored
  v = join(v, dpp<0x140>(v));  // of sixteen
  return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_max(float v) {
  return over_wave(v, [](float p, float q) { return __builtin_fmaxf(p, q); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return over_wave(v, [](float p, float q) { return p + q; });
}
// The largest over groups of G lanes, in all of them.
template <int G>
__device__ __forceinline__ float group_max(float v) {
  if (G >= 2) v = __builtin_fmaxf(v, dpp<0xB1>(v));
  if (G >= 4) v = __builtin_fmaxf(v, dpp<0x4E>(v));
  if (G >= 8) v = __builtin_fmaxf(v, dpp<0x141>(v));
  return v;
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
#pragma unroll
  for (int step = 32; step; step /= 2) {
    const unsigned long long o = (unsigned long long)__shfl_xor((unsigned)(v >> 32), step) << 32 | __shfl_xor((unsigned)v, step);
    v = o > v ? o : v;
  }
  return v;
}

constexpr float kLog2E = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kLowest = -3.402823466e38f;  // where maxima start: minus infinity less this is minus infinity, no NaN

constexpr float kNoPower = -1e4f;          // 2 to it is 0, and so is its product with it; that of minus infinity would be NaN (maximum keeps a NaN)

// Maximum and sums of part of a row: s = sum 2^t, w = sum t 2^t, t = (x - m) log2 e.
struct RowSums {
  float m, s, w;
};
// Of sums whose maxima differ, one per lane.
__device__ __forceinline__ RowSums join_sums(RowSums p) {
  const float m = wave_max(p.m), t = __builtin_fmaxf((p.m - m) * kLog2E, kNoPower);
  const float c = __builtin_amdgcn_exp2f(t);
  return {m, wave_sum(c * p.s), wave_sum(c * __builtin_fmaf(t, p.s, p.w))};
}

// Results of a row from its sums (one lane), and what a log probability is made of.
struct RowNorm {
  float base, log_s;
  __device__ __forceinline__ RowNorm(RowSums r) : base(r.m), log_s(logf(r.s)) {}
  __device__ __forceinline__ float log_prob(float x) const { return x == -__builtin_inff() ? x : (x - base) - log_s; }
};
template <typename AT>
__device__ __forceinline__ void row_results(const ScoresArgs& a, long long r, long long target, RowSums sums) {
  const RowNorm norm(sums);
  if (a.norm) a.norm[2 * r] = norm.base, a.norm[2 * r + 1] = norm.log_s;
  if (a.log_prob) a.log_prob[r] = target < a.V ? norm.log_prob(load_f32((const AT*)a.logits + r * a.ld + target)) : __builtin_nanf("");
  if (a.entropy) a.entropy[r] = sums.s == 0.f ? 0.f : norm.log_s - kLn2 * (sums.w / sums.s);
}
// ... of a row without a token, by `threads` threads
__device__ __forceinline__ void no_row(const ScoresArgs& a, long long r, int thread, int threads) {
  if (thread == 0) {
    if (a.log_prob) a.log_prob[r] = 0.f;
    if (a.norm) a.norm[2 * r] = a.norm[2 * r + 1] = 0.f;
    if (a.entropy) a.entropy[r] = 0.f;
  }
  for (int k = thread; k < a.top_k; k += threads) {
    a.top_log_prob[r * a.top_k + k] = -__builtin_inff();
    a.top_ids[r * a.top_k + k] = -1;
  }
}
// Alternative number `rank` of a row, or of a piece of it.
__device__ __forceinline__ void put_alternative(const ScoresArgs& a, long long r, int split, int rank, unsigned long long q, const RowNorm& norm) {
  if (a.splits > 1) {
    a.part_top[(r * a.splits + split) * a.top_k + rank] = q;
  } else {
    a.top_log_prob[r * a.top_k + rank] = norm.log_prob(logit_of(q));
    a.top_ids[r * a.top_k + rank] = (int64_t)(unsigned)~(unsigned)q;
  }
}

// W wavefronts per row or piece of one (W = 1: four rows per workgroup), E logits per lane, all in registers.
constexpr int kCandidates = 256;
constexpr int kMaxSegment = 16 * 64 * 32;
constexpr long long kMaxTokens = 1 << 26;  // (pieces are a multiple of 8 long: with many more of them nothing would be left for the last)
template <typename AT, int W, int E, bool TOP>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_token_scores(ScoresArgs a) {
  constexpr int R = W == 1 ? 4 : 1;                  // rows per workgroup
  constexpr int GROUPS = W == 1 ? 64 : 128;          // of lanes, whose maxima bound the alternatives from below
  constexpr int GROUP = 64 * W / GROUPS;
  __shared__ float sums_of[R][W][4];
  __shared__ float group_of[TOP ? R : 1][TOP ? GROUPS : 1];
  __shared__ unsigned long long list_of[TOP ? R : 1][TOP ? kCandidates : 1];
  __shared__ int listed_of[R];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, sub = W == 1 ? threadIdx.x >> 6 : 0, thread = wave * 64 + lane;
  const long long item = blockIdx.x * (long long)R + sub;
  if (W == 1 && item >= a.rows) return;
  const long long r = a.splits > 1 ? (unsigned)item / (unsigned)a.splits : item;
  const int split = a.splits > 1 ? (int)(item - r * a.splits) : 0;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    if (a.splits == 1) no_row(a, r, thread, 64 * W);
    return;
  }
  const AT* row = (const AT*)a.logits + r * a.ld;
  const long long v0 = split * a.segment, v1 = v0 + a.segment < a.V ? v0 + a.segment : a.V;
  const float inf = __builtin_inff();
  float x[E];
  int index[W == 1 ? 1 : E / 8];  // of a lane's eight, from v0 on
  if constexpr (W == 1) {
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = k * 64 + lane < v1 ? load_f32(row + k * 64 + lane) : -inf;
    index[0] = lane;
  } else {
    // Eight neighbours are one load; those that reach past the end of the row are its last eight (there are more than eight), of which the
    // ones that an earlier lane has are left out.
    const int count = (int)(v1 - v0);
    Eight<AT> q[E / 8];
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      index[j] = (j * 64 * W + thread) * 8;
      const long long at = v0 + index[j];
      q[j].load(row + (at < a.V - 8 ? at : a.V - 8));
    }
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      float v[8];
      q[j].get(v);
      if (__any(index[j] + 8 > count)) {
        const int from = index[j], begin = v0 + from < a.V - 8 ? from : (int)(a.V - 8 - v0);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = begin + k >= from && begin + k < count ? v[k] : -inf;
        index[j] = begin;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[8 * j + k] = v[k];
    }
  }
  auto index_of = [&](int k) { return (unsigned)(v0 + (W == 1 ? k * 64 + index[0] : index[k / 8] + k % 8)); };

  float most = kLowest;
#pragma unroll
  for (int k = 0; k < E; ++k) most = __builtin_fmaxf(most, x[k]);
  const float m = wave_max(most);
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const float t = __builtin_elementwise_maximum((x[k] - m) * kLog2E, kNoPower), e = __builtin_amdgcn_exp2f(t);
    s += e;
    w = __builtin_fmaf(t, e, w);
  }
  RowSums sums{m, wave_sum(s), wave_sum(w)};
  if constexpr (W > 1) {
    if (lane == 0) sums_of[0][wave][0] = sums.m, sums_of[0][wave][1] = sums.s, sums_of[0][wave][2] = sums.w;
    if (TOP) {
      const float g = group_max<GROUP>(most);
      if (lane % GROUP == 0) group_of[0][thread / GROUP] = g;
      if (thread == 0) listed_of[0] = 0;
    }
    __syncthreads();
    sums = lane < W ? RowSums{sums_of[0][lane % W][0], sums_of[0][lane % W][1], sums_of[0][lane % W][2]} : RowSums{kLowest, 0.f, 0.f};
    sums = join_sums(sums);
  }
  if (thread == 0) {
    if (a.splits > 1) {
      float* part = a.part + (r * a.splits + split) * 4;
      part[0] = sums.m, part[1] = sums.s, part[2] = sums.w;
    } else {
      row_results<AT>(a, r, target, sums);
    }
  }
  if constexpr (TOP) {
    const RowNorm norm(sums);
    unsigned long long* list = list_of[sub];
    int* listed = &listed_of[sub];
    bool found = false;
    if (sums.s > 0.f && sums.s < inf) {
      // A bound from below: the top_k-th largest of the groups' maxima, found bit by bit from the top (bfloat16 has 16).
      unsigned low0, low1 = 0;
      if constexpr (W == 1) {
        low0 = order_of(most);
        if (lane == 0) *listed = 0;
      } else {
        low0 = order_of(group_of[0][lane]);
        low1 = order_of(group_of[0][64 + lane]);
      }
      unsigned bound = 0;
#pragma unroll 1
      for (unsigned bit = 0x80000000u; bit > (sizeof(AT) == 2 ? 0x8000u : 0u); bit >>= 1) {
        const unsigned next = bound | bit;
        const int over = __popcll(__ballot(low0 >= next)) + (W == 1 ? 0 : __popcll(__ballot(low1 >= next)));
        if (over >= a.top_k) bound = next;
      }
      const float at_least = logit_of((unsigned long long)bound << 32);
      // What reaches it is listed, in any order, and every listed one finds its rank among them.
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (x[k] >= at_least) {
          const int at = atomicAdd(listed, 1);
          if (at < kCandidates) list[at] = alternative(x[k], index_of(k));
        }
      if constexpr (W > 1)
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int n = *(volatile int*)listed;
      found = n >= a.top_k && n <= kCandidates;
      if (found)
        for (int j = thread; j < n; j += 64 * W) {
          const unsigned long long mine = list[j];
          int rank = 0;
          for (int o = 0; o < n; ++o) rank += list[o] > mine;
          if (rank < a.top_k) put_alternative(a, r, split, rank, mine, norm);
        }
    }
    if (!found) {
      // More equal logits than the list holds, fewer finite ones than wanted, a NaN: the best one of all, and again.  Every lane knows its best
      // one; whose turn it was looks for its next.  (What a lane holds past the end, or of another lane's, is minus infinity at the last indices
      // of the row: it comes after more real ones than are ever wanted.)
      if constexpr (W > 1) __syncthreads();  // (the list is read no more)
      unsigned long long last = ~0ull, mine = 0;
      auto look = [&]() {
        mine = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const unsigned long long q = alternative(x[k], index_of(k));
          const bool real = W == 1 ? k * 64 + lane < v1 : true;
          if (q < last && q > mine && real) mine = q;
        }
      };
      look();
#pragma unroll 1
      for (int k = 0; k < a.top_k; ++k) {
        unsigned long long best = wave_max(mine);
        if constexpr (W > 1) {
          if (lane == 0) list[(k & 1) * W + wave] = best;
          __syncthreads();
          best = wave_max(list[(k & 1) * W + lane % W]);
        }
        if (thread == 0) put_alternative(a, r, split, k, best, norm);
        if (mine == best) {
          last = best;
          look();
        }
      }
    }
  }
}

// The pieces of a row joined.  One workgroup per row; the alternatives of the pieces are sorted lists, and every one finds its rank in all of them.
constexpr int kJoinInLds = 4096;
template <typename AT>
__global__ __launch_bounds__(256) void k_token_scores_join(ScoresArgs a) {
  __shared__ unsigned long long held[kJoinInLds];
  const long long r = blockIdx.x;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    no_row(a, r, threadIdx.x, 256);
    return;
  }
  const int lane = threadIdx.x & 63;
  RowSums sums{kLowest, 0.f, 0.f};
  for (int j = lane; j < a.splits; j += 64) {  // (lanes' own pieces one after the other, in every wavefront alike)
    const float* p = a.part + (r * a.splits + j) * 4;
    const RowSums next{p[0], p[1], p[2]};
    const float top = __builtin_fmaxf(sums.m, next.m);
    const float t0 = __builtin_fmaxf((sums.m - top) * kLog2E, kNoPower), t1 = __builtin_fmaxf((next.m - top) * kLog2E, kNoPower);
    const float c0 = __builtin_amdgcn_exp2f(t0), c1 = __builtin_amdgcn_exp2f(t1);
    sums = {top, c0 * sums.s + c1 * next.s, c0 * __builtin_fmaf(t0, sums.s, sums.w) + c1 * __builtin_fmaf(t1, next.s, next.w)};
  }
  sums = join_sums(sums);
  if (threadIdx.x == 0) row_results<AT>(a, r, target, sums);
  if (a.top_k == 0) return;
  const RowNorm norm(sums);
  const long long n = (long long)a.splits * a.top_k;
  const unsigned long long* all = a.part_top + r * n;
  if (n <= kJoinInLds) {
    for (int j = threadIdx.x; j < n; j += 256) held[j] = all[j];
    __syncthreads();
  }
  for (long long j = threadIdx.x; j < n; j += 256) {
    const unsigned long long mine = n <= kJoinInLds ? held[j] : all[j];
    long long rank = 0;
    for (int p = 0; p < a.splits && rank < a.top_k; ++p) {
      int low = 0, high = a.top_k;  // how many of piece p are larger
      while (low < high) {
        const int mid = (low + high) / 2;
        const unsigned long long q = n <= kJoinInLds ? held[p * a.top_k + mid] : all[(long long)p * a.top_k + mid];
        if (q > mine)
          low = mid + 1;
        else
          high = mid;
      }
      rank += low;
    }
    if (rank < a.top_k && mine) {
      a.top_log_prob[r * a.top_k + rank] = norm.log_prob(logit_of(mine));
      a.top_ids[r * a.top_k + rank] = (int64_t)(unsigned)~(unsigned)mine;
    }
  }
}

// D = p (A + B t), plus d_log_prob at the target; t = log2 p.  ROW: a wavefront per row, four rows per workgroup; else a workgroup per piece of
// kBwdPiece logits of a row.
constexpr int kBwdPiece = 8192;
template <typename AT, bool ROW>
__global__ __launch_bounds__(256) void k_token_scores_bwd(ScoresArgs a) {
  constexpr int THREADS = ROW ? 64 : 256, N = ROW ? 1 : kBwdPiece / (256 * 8);
  const int thread = ROW ? threadIdx.x & 63 : threadIdx.x;
  const long long item = ROW ? blockIdx.x * 4ll + (threadIdx.x >> 6) : blockIdx.x;
  if (ROW && item >= a.rows) return;
  const long long r = ROW ? item : (unsigned)item / (unsigned)a.splits, v0 = ROW ? 0 : (item - r * a.splits) * kBwdPiece;
  const long long v1 = ROW ? a.V : (v0 + kBwdPiece < a.V ? v0 + kBwdPiece : a.V);
  const AT* x = (const AT*)a.logits + r * a.ld;
  AT* D = (AT*)a.D + r * a.V;
  const long long target = a.targets ? a.targets[r] : 0;
  const float base = a.norm[2 * r], log_s = a.norm[2 * r + 1];
  const float g = a.d_log_prob ? a.d_log_prob[r] : 0.f, ge = a.d_entropy ? a.d_entropy[r] : 0.f, h = a.d_entropy ? a.entropy[r] : 0.f;
  const bool none = target < 0 || log_s == -__builtin_inff();
  const float A = a.targets && target >= a.V ? __builtin_nanf("") : -__builtin_fmaf(ge, h, g), B = -ge * kLn2, c = -log_s * kLog2E;
  auto one = [&](float v) {
    const float t = __builtin_elementwise_maximum(__builtin_fmaf(v - base, kLog2E, c), kNoPower);
    return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(B, t, A);
  };
  const bool known = a.targets != nullptr && !none;
  for (long long from = v0; from < v1; from += (long long)THREADS * 8 * N) {
    const long long first = from + thread * 8;
    if (from + (long long)THREADS * 8 * N <= v1) {
      Eight<AT> q[N];
      if (!none) {
#pragma unroll
        for (int j = 0; j < N; ++j) q[j].load(x + first + j * THREADS * 8);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const long long at = first + j * THREADS * 8;
        float v[8];
        if (none) {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = 0.f;
        } else {
          q[j].get(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = one(v[k]);
          if (known && target >= at && target < at + 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += target == at + k ? g : 0.f;
          }
        }
        q[j].set(v);
        q[j].store(D + at);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < N; ++j) {
        const long long at = first + j * THREADS * 8;
        if (at + 8 <= v1) {
          Eight<AT> q;
          float v[8];
          if (!none) q.load(x + at);
          q.get(v);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = none ? 0.f : one(v[k]) + (known && target == at + k ? g : 0.f);
          q.set(v);
          q.store(D + at);
        } else {
          for (long long k = at; k < v1; ++k) store_f32(D + k, none ? 0.f : one(load_f32(x + k)) + (known && target == k ? g : 0.f));
        }
      }
    }
  }
}

}  // namespace rtn
