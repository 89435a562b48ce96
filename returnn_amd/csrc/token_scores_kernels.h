// gfx950 kernels of log probabilities of tokens, entropy and alternatives, and of their gradient.
//
//   lse = m + log s,  s = sum e^(x-m),  log_prob = x_target - lse,  entropy = log s - w / s,  w = sum (x-m) e^(x-m)
//   D_v = d_log_prob (1[v = target] - p_v) - d_entropy p_v (log p_v + entropy)
#pragma once

#include <type_traits>

#include "sequence_common.h"

namespace rtn {

constexpr int kMaxAlternatives = 64;

struct ScoresArgs {
  const void* logits;
  long long ld;
  const int64_t* targets;
  long long rows;
  int V;
  int top_k;
  float *log_prob, *norm, *entropy, *top_log_prob;
  int64_t* top_ids;
  const float *d_log_prob, *d_entropy;
  void* D;
  int splits;          // pieces of a row
  int segment;         // logits of a piece
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
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
#pragma unroll
  for (int step = 32; step; step /= 2) {
    const unsigned long long o = (unsigned long long)__shfl_xor((unsigned)(v >> 32), step) << 32 | __shfl_xor((unsigned)v, step);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ unsigned wave_min(unsigned v) {
  auto other = [&](auto ctrl) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, true); };
  auto least = [](unsigned p, unsigned q) { return p < q ? p : q; };
  v = least(v, other(std::integral_constant<int, 0xB1>()));  // (as in over_wave)
  v = least(v, other(std::integral_constant<int, 0x4E>()));
  v = least(v, other(std::integral_constant<int, 0x141>()));
  v = least(v, other(std::integral_constant<int, 0x140>()));
  auto at = [&](int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); };
  return least(least(at(0), at(16)), least(at(32), at(48)));
}

constexpr float kLog2E = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kLowest = -3.402823466e38f;  // where maxima start: minus infinity less this is minus infinity, no NaN

constexpr float kNothing = -1e30f;         // 2^(it less a logit) is 0, and so is its product with it
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

// ... of the 16 lanes of a quarter, in all of them.
template <typename F>
__device__ __forceinline__ float over_quarter(float v, F join) {
  v = join(v, dpp<0xB1>(v));
  v = join(v, dpp<0x4E>(v));
  v = join(v, dpp<0x141>(v));
  return join(v, dpp<0x140>(v));
}
// The k-th largest of what the 16 lanes of a quarter have, k = 1 to 16, in all of them.
template <int R>
__device__ __forceinline__ int larger_in_quarter(float v) {
  if constexpr (R == 0)
    return 0;
  else
    return larger_in_quarter<R - 1>(v) + (dpp<0x120 + R>(v) > v);  // (the lane R further, around)
}
__device__ __forceinline__ float kth_of_quarter(float v, int k) {
  return over_quarter(larger_in_quarter<15>(v) < k ? v : __builtin_inff(), [](float x, float y) { return __builtin_fminf(x, y); });
}
__device__ __forceinline__ RowSums join_quarter(RowSums p) {
  auto add = [](float x, float y) { return x + y; };
  const float m = over_quarter(p.m, [](float x, float y) { return __builtin_fmaxf(x, y); }), t = __builtin_fmaxf((p.m - m) * kLog2E, kNoPower);
  const float c = __builtin_amdgcn_exp2f(t);
  return {m, over_quarter(c * p.s, add), over_quarter(c * __builtin_fmaf(t, p.s, p.w), add)};
}

// Results of a row from its sums (one lane), and what a log probability is made of.
struct RowNorm {
  float base, log_s;
  RowNorm() = default;
  __device__ __forceinline__ RowNorm(RowSums r) : base(r.m), log_s(logf(r.s)) {}
  // (minus infinity of a token that is not allowed, but not beside a NaN)
  __device__ __forceinline__ float log_prob(float x) const { return x == -__builtin_inff() && log_s == log_s ? x : (x - base) - log_s; }
};
template <typename AT>
__device__ __forceinline__ RowNorm row_results(const ScoresArgs& a, long long r, long long target, RowSums sums) {
  const RowNorm norm(sums);
  if (a.norm) a.norm[2 * r] = norm.base, a.norm[2 * r + 1] = norm.log_s;
  if (a.log_prob) a.log_prob[r] = target < a.V ? norm.log_prob(load_f32((const AT*)a.logits + r * a.ld + target)) : __builtin_nanf("");
  if (a.entropy) a.entropy[r] = sums.s == 0.f ? 0.f : norm.log_s - kLn2 * (sums.w / sums.s);
  return norm;
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

// The sum over 16 neighbouring lanes, in all of them.
__device__ __forceinline__ int quarter_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, true);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, true);
}
// How many of the n of a list are larger than `mine`, of which 16 neighbouring lanes look at every 16th: the same in all of them.  (One lane by itself goes through
// a chain of look-ups and 64-bit comparisons: of 44, which is usual for 12 alternatives, 3000 clocks, a fifth of the kernel.)
__device__ __forceinline__ int rank_in(const unsigned long long* list, int n, unsigned long long mine, int lane) {
  int rank = 0;
#pragma unroll 4
  for (int o = lane & 15; o < n; o += 16) rank += list[o] > mine;
  return quarter_sum(rank);
}

// Sums and alternatives: W wavefronts per row or piece of one (W = 1: four rows per workgroup), E logits per lane, all in registers.
// For few rows bound by latency: 12 rows of 32000 bf16 with 12 alternatives 6.8 us, with 1 6.0, the sums alone 4.8; for many by memory and the lists' barriers:
// 3000 such rows 52 us (192 MB, 3.7 TB/s), the sums alone 42.
constexpr int kCandidates = 512;
constexpr int kCoarse = 48;  // alternatives up to which 64 groups are enough
constexpr int kMaxSegment = 16 * 64 * 32;
constexpr long long kMaxTokens = 1 << 26;  // (pieces are a multiple of 8 long: with many more of them nothing would be left for the last)
template <typename AT, int W, int E>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_token_scores_top(ScoresArgs a) {
  constexpr int R = W == 1 ? 4 : 1;            // rows per workgroup
  constexpr int LANES = W == 1 ? 1 : W / 4;  // that have one of 256 groups
  constexpr bool SINGLE = E == 8 && W == 1;  // logits one by one, not by eights, of which there have to be some
  __shared__ float sums_of[R][W][4];
  __shared__ alignas(16) float most_of[W][64];
  __shared__ unsigned long long list_of[R][kCandidates];
  __shared__ int listed_of[R];
  __shared__ float norm_of[R][2];
  __shared__ int larger_of[64];
  __shared__ float bound_of[W];
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
  const int v0 = split * a.segment, v1 = v0 + a.segment < a.V ? v0 + a.segment : a.V;
  const float inf = __builtin_inff();
  float x[E];
  // (where the eight number j of this lane begins, and where its logits are read: the last ones of the row are its last eight -- there are more than
  // eight --, of which the ones that an earlier lane has are left out)
  auto own = [&](int j) { return v0 + (j * 64 * W + thread) * 8; };
  auto read = [&](int j) { return own(j) < a.V - 8 ? own(j) : a.V - 8; };
  if constexpr (SINGLE) {
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = k * 64 + lane < v1 ? load_f32(row + k * 64 + lane) : -inf;
  } else {
    Eight<AT> q[E / 8];
#pragma unroll
    for (int j = 0; j < E / 8; ++j) q[j].load(row + read(j));
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      float v[8];
      q[j].get(v);
      if (__any(own(j) + 8 > v1)) {
        const int from = own(j) - read(j), to = v1 - read(j);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = k >= from && k < to ? v[k] : -inf;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) x[8 * j + k] = v[k];
    }
  }

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
  bool finite = sums.s < inf;  // (neither a NaN nor an infinity in the row)
  float group = most;
  if constexpr (W == 1) {
    if (lane == 0) listed_of[sub] = 0;
  } else {
    if (a.top_k > kCoarse) {
      if (W >= 8) group = __builtin_fmaxf(group, dpp<0xB1>(group));
      if (W == 16) group = __builtin_fmaxf(group, dpp<0x4E>(group));
      if (lane % LANES == 0) (&most_of[0][0])[thread / LANES] = group;
    } else {
      most_of[wave][lane] = most;
    }
    if (lane == 0) sums_of[0][wave][0] = sums.m, sums_of[0][wave][1] = sums.s, sums_of[0][wave][2] = sums.w;
    if (thread == 0) listed_of[0] = 0;
    if (wave == 0) larger_of[lane] = 0;
    __syncthreads();
    sums = lane < W ? RowSums{sums_of[0][lane % W][0], sums_of[0][lane % W][1], sums_of[0][lane % W][2]} : RowSums{kLowest, 0.f, 0.f};
    finite = !__any(!(sums.s < inf));
  }
  auto meet = [&]() {
    if constexpr (W > 1)
      __syncthreads();
    else
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  unsigned long long* list = list_of[sub];
  int* listed = &listed_of[sub];
  int n = 0;
  float bound = kLowest;
  // Lists what reaches the bound, in any order.
  auto make_list = [&]() {
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      unsigned hits = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) hits |= x[8 * j + k] >= bound ? 1u << k : 0u;
      if (hits) {
        int at = atomicAdd(listed, __popc(hits));
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (hits >> k & 1u) {
            if (at < kCandidates) list[at] = alternative(x[8 * j + k], (unsigned)(SINGLE ? k * 64 + lane : read(j) + k));
            ++at;
          }
      }
    }
    meet();
    n = *(volatile int*)listed;
  };
  if (finite) {
    // A bound from below: the logits are dealt to 16 groups, to 64 for more than 16 alternatives or (unless the row has one wavefront) to 256 for more than
    // kCoarse, and the top_k-th largest of the groups' maxima is reached by top_k logits at least.  What reaches it is listed (for 1, 12, 20, 64 alternatives
    // about 1, 21, 24, 74) and finds its rank in the list.  (The top_k-th largest of 128 maxima, found bit by bit, took longer than all the rest: one row of
    // 32768 float32 with 12 alternatives 9.6 us, with this 6.3.  64 groups for 64 alternatives: 12 rows of 32000 bf16 16.5 us, with 256 9.1; 16 groups
    // and 64 for 5: 9000 rows of 500 12.5 and 17.1.)  The groups are the wavefronts, or what neighbouring lanes have, of all wavefronts or of one.
    if constexpr (W > 1) {
      if ((W < 16 || a.top_k > 16) && a.top_k <= kCoarse) {
#pragma unroll
        for (int o = 0; o < W; ++o) group = __builtin_fmaxf(group, most_of[o][lane]);
      }
    }
    if (a.top_k <= 16) {
      if (W == 16) {
        group = sums.m;
      } else {
        group = __builtin_fmaxf(group, dpp<0xB1>(group));
        group = __builtin_fmaxf(group, dpp<0x4E>(group));
        group = __shfl(group, lane * 4 & 63);
      }
      bound = lane_of(kth_of_quarter(group, a.top_k), 0);
    } else if (W > 1 && a.top_k > kCoarse) {
      const float* maxima = &most_of[0][0];
      const int part = thread % LANES;
      group = maxima[thread / LANES];
      int larger = 0;  // (a group's lanes look at a part of the others each, from different banks on)
#pragma unroll 4
      for (int o = 0; o < 256 / LANES; o += 4) {
        const float* four = maxima + part * (256 / LANES) + (o + 4 * part) % (256 / LANES);
#pragma unroll
        for (int k = 0; k < 4; ++k) larger += four[k] > group;
      }
      if (LANES > 1) larger += __builtin_amdgcn_update_dpp(0, larger, 0xB1, 0xF, 0xF, true);
      if (LANES > 2) larger += __builtin_amdgcn_update_dpp(0, larger, 0x4E, 0xF, 0xF, true);
      bound = wave_max(larger < a.top_k ? -group : -inf);
      if (lane == 0) bound_of[wave] = bound;
      __syncthreads();
      bound = -wave_max(lane < W ? bound_of[lane % W] : -inf);
    } else {
      int larger = 0;  // (every wavefront looks at some of the others)
#pragma unroll 4
      for (int o = 0; o < 64 / W; ++o) larger += __shfl(group, lane + wave * (64 / W) + o & 63) > group;
      if constexpr (W > 1) {
        atomicAdd(&larger_of[lane], larger);
        __syncthreads();
        larger = larger_of[lane];
      }
      bound = -wave_max(larger < a.top_k ? -group : -inf);
    }
  }
  RowNorm norm;
  if (wave == 0) {  // (the others are at their lists)
    if constexpr (W > 1) sums = join_quarter(sums);
    if (lane == 0) {
      if (a.splits > 1) {
        float* part = a.part + (r * a.splits + split) * 4;
        part[0] = sums.m, part[1] = sums.s, part[2] = sums.w;
      } else {
        norm = row_results<AT>(a, r, target, sums);
      }
      norm_of[sub][0] = norm.base, norm_of[sub][1] = norm.log_s;
    }
  }
  if (finite) {
    make_list();
    if (!SINGLE && n > kCandidates) {
      // Too many: the largest bound that top_k lanes still reach, to within a 4096th of what is in question.
      float high = W > 1 ? wave_max(lane < W ? sums_of[0][lane % W][0] : kLowest) : sums.m;
#pragma unroll 1
      for (int step = 0; step < 12; ++step) {
        const float mid = 0.5f * bound + 0.5f * high;
        meet();  // (everyone has read what is written here)
        if (thread == 0) *listed = 0;
        meet();
        const int reach = __popcll(__ballot(most >= mid));
        if (lane == 0) atomicAdd(listed, reach);
        meet();
        if (*(volatile int*)listed >= a.top_k)
          bound = mid;
        else
          high = mid;
      }
      meet();
      if (thread == 0) *listed = 0;
      meet();
      make_list();
    }
  } else {
    meet();
  }
  norm.base = norm_of[sub][0], norm.log_s = norm_of[sub][1];
  // (fewer than wanted, but all that are not minus infinity, are also good)
  if (finite && n <= kCandidates && (n >= a.top_k || bound == kLowest)) {
    // (by 16 lanes each where there are many, see rank_in; but that is more work, which counts where rows are short and many)
    if constexpr (W >= 8) {
      for (int j = thread >> 4; j < n; j += 4 * W) {
        const unsigned long long mine = list[j];
        const int rank = rank_in(list, n, mine, lane);
        if ((lane & 15) == 0 && rank < a.top_k) put_alternative(a, r, split, rank, mine, norm);
      }
    } else {
      for (int j = thread; j < n; j += 64 * W) {
        const unsigned long long mine = list[j];
        int rank = 0;
#pragma unroll 8
        for (int o = 0; o < n; ++o) rank += list[o] > mine;
        if (rank < a.top_k) put_alternative(a, r, split, rank, mine, norm);
      }
    }
    // The first ones that are minus infinity: among the first top_k of the row, then, there are as many as are wanted.
    if (wave == 0)
      for (int v = v0; n < a.top_k && v < v1; v += 64) {
        const bool is = v + lane < v1 && load_f32(row + v + lane) == -inf;
        const unsigned long long all = __ballot(is);
        const int rank = n + __popcll(all & ((1ull << lane) - 1));
        if (is && rank < a.top_k) put_alternative(a, r, split, rank, alternative(-inf, (unsigned)(v + lane)), norm);
        n += __popcll(all);
      }
    return;
  }
  // More equal logits than the list holds, or a NaN: the best one of all, and again.  Every lane knows its best one; whose turn it was looks for
  // its next.  (What a lane holds of another lane's it skips.)
  meet();  // (the list is read no more)
  unsigned long long last = ~0ull, mine = 0;
#pragma unroll 1
  for (int k = -1; k < a.top_k; ++k) {
    unsigned long long best = last;
    if (k >= 0) {
      best = wave_max(mine);
      if constexpr (W > 1) {
        if (lane == 0) list[(k & 1) * W + wave] = best;
        __syncthreads();
        best = wave_max(list[(k & 1) * W + lane % W]);
      }
      if (thread == 0) put_alternative(a, r, split, k, best, norm);
    }
    if (k < 0 || mine == best) {
      last = best;
      mine = 0;
#pragma unroll 8
      for (int j = 0; j < E; ++j) {
        const int at = SINGLE ? v0 + j * 64 + lane : own(j >> 3) + (j & 7);
        if (at < v1) {
          const unsigned long long q = alternative(load_f32(row + at), (unsigned)at);
          if ((k < 0 || q < last) && q > mine) mine = q;  // (nothing is larger than a NaN at index 0)
        }
      }
    }
  }
}

// Short rows of which there are many: 16 lanes per row, eight neighbouring logits of a lane at a time (there are eight at least).  The bound is as above, with the
// 16 lanes as groups; where it is none, or the row has a NaN or an infinity, all logits are listed.  One wavefront per row spends most of its time on what is the
// same for a row of any length (us, with one / with this: 70000 rows of 96 bf16, sums 25.1 / 6.7, with 5 alternatives 40.8 / 13.5; of 256 25.8 / 10.5, 45.5 / 20.5).
template <typename AT, int E>
__global__ __launch_bounds__(256) void k_token_scores_short(ScoresArgs a) {
  __shared__ unsigned long long list_of[16][16 * E];
  __shared__ int listed_of[16];
  const int lane = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const long long r = blockIdx.x * 16ll + sub;
  if (r >= a.rows) return;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    no_row(a, r, lane, 16);
    return;
  }
  const AT* row = (const AT*)a.logits + r * a.ld;
  const float inf = __builtin_inff();
  auto own = [&](int j) { return (j * 16 + lane) * 8; };
  auto read = [&](int j) { return own(j) < a.V - 8 ? own(j) : a.V - 8; };
  float x[E], most = kLowest;
  Eight<AT> q[E / 8];
#pragma unroll
  for (int j = 0; j < E / 8; ++j) q[j].load(row + read(j));
#pragma unroll
  for (int j = 0; j < E / 8; ++j) {
    float v[8];
    q[j].get(v);
    const int from = own(j) - read(j);  // (what an earlier lane has is left out)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[8 * j + k] = k >= from ? v[k] : -inf;
      most = __builtin_fmaxf(most, x[8 * j + k]);
    }
  }
  auto add = [](float p, float q) { return p + q; };
  const float m = over_quarter(most, [](float p, float q) { return __builtin_fmaxf(p, q); });
  float s = 0.f, w = 0.f;
#pragma unroll
  for (int k = 0; k < E; ++k) {
    const float t = __builtin_elementwise_maximum((x[k] - m) * kLog2E, kNoPower), e = __builtin_amdgcn_exp2f(t);
    s += e;
    w = __builtin_fmaf(t, e, w);
  }
  const RowSums sums{m, over_quarter(s, add), over_quarter(w, add)};
  if (lane == 0) {
    row_results<AT>(a, r, target, sums);
    listed_of[sub] = 0;
  }
  if (a.top_k == 0) return;
  const RowNorm norm(sums);
  const float bound = a.top_k <= 16 ? kth_of_quarter(most, a.top_k) : kLowest;
  const bool all = !(sums.s < inf) || bound <= kLowest;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  unsigned long long* list = list_of[sub];
#pragma unroll
  for (int j = 0; j < E / 8; ++j) {
    const int from = own(j) - read(j);
    unsigned hits = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) hits |= k >= from && (all || x[8 * j + k] >= bound) ? 1u << k : 0u;
    if (hits) {
      int at = atomicAdd(&listed_of[sub], __popc(hits));
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (hits >> k & 1u) list[at++] = alternative(x[8 * j + k], (unsigned)(read(j) + k));
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int n = *(volatile int*)&listed_of[sub];
  for (int j = lane; j < n; j += 16) {
    const unsigned long long mine = list[j];
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < n; ++o) rank += list[o] > mine;
    if (rank < a.top_k) put_alternative(a, r, 0, rank, mine, norm);
  }
}

// Sums without alternatives, read as they come: W wavefronts per row or piece of one (W = 1: four rows per workgroup), U times eight logits per
// lane in flight.  The wavefront's reference, which stands for the maximum, is that of the first 512 logits among which one is above kNothing (of tokens that are
// not allowed, minus infinity or the type's lowest value, nothing is left beside it).  Where a lane's sum passes kRise, the logits that are held are added
// once more, relative to the largest so far: so no logit is more than 22 above its reference, and sums of all lanes, wavefronts and pieces are far from what
// float32 ends at.  (A maximum of every logit beforehand would be one instruction more for each; this is one for 32 of them.)  Where the sums are not finite all the same, or
// there is no such reference, the wavefront takes them again, with the true maximum.
// Bound by memory: 4096 rows of 32000 bf16 53 us (262 MB, 4.95 TB/s), the same where the first 2048 logits lie 60 lower.  (Products of minus infinity left to be NaN
// and found afterwards: 1 us less, but 262 where tokens are masked.)
constexpr float kRise = 0x1p32f;
template <typename AT, int W, bool ENTROPY>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void k_token_scores(ScoresArgs a) {
  constexpr int R = W == 1 ? 4 : 1, U = 4;
  __shared__ float sums_of[W][4];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, thread = wave * 64 + lane;
  const long long item = blockIdx.x * (long long)R + (W == 1 ? threadIdx.x >> 6 : 0);
  if (W == 1 && item >= a.rows) return;
  const long long r = a.splits > 1 ? (unsigned)item / (unsigned)a.splits : item;
  const int split = a.splits > 1 ? (int)(item - r * a.splits) : 0;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    if (a.splits == 1) no_row(a, r, thread, 64 * W);
    return;
  }
  const AT* row = (const AT*)a.logits + r * a.ld;
  const int v0 = split * a.segment, v1 = v0 + a.segment < a.V ? v0 + a.segment : a.V;
  RowSums sums{kLowest, 0.f, 0.f};
  const bool vector = a.V >= 8;
  bool referred = false;
#pragma unroll 1
  for (int from = v0; vector && from + wave * 512 < v1; from += 512 * W * U) {
    Eight<AT> q[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int at = from + (j * 64 * W + thread) * 8;
      q[j].load(row + (at < a.V - 8 ? at : a.V - 8));
    }
    const RowSums before = sums;
    auto first = [&](int j) { return from + (j * 64 * W + wave * 64) * 8; };  // of the wavefront's logits
    auto get = [&](int j, float (&v)[8]) {
      q[j].get(v);
      if (first(j) + 512 > v1) {  // see above: the last eight of the row, those of an earlier lane left out
        const int mine = first(j) + lane * 8, begin = mine < a.V - 8 ? mine : a.V - 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = begin + k >= mine && begin + k < v1 ? v[k] : kNothing;
      }
    };
    auto add = [&](const float (&v)[8]) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float t = (v[k] - sums.m) * kLog2E;
        if (ENTROPY) t = __builtin_elementwise_maximum(t, kNoPower);  // (a product of minus infinity with 0 would be NaN)
        const float e = __builtin_amdgcn_exp2f(t);
        sums.s += e;
        if (ENTROPY) sums.w = __builtin_fmaf(t, e, sums.w);
      }
    };
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (first(j) >= v1) break;
      float v[8];
      get(j, v);
      if (!referred) {
        float most = kLowest;
#pragma unroll
        for (int k = 0; k < 8; ++k) most = __builtin_fmaxf(most, v[k]);
        sums = {wave_max(most), 0.f, 0.f};
        referred = sums.m > kNothing;
      }
      add(v);
    }
    if (__any(sums.s > kRise)) {
      float most = before.m;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (first(j) >= v1) break;
        float v[8];
        get(j, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) most = __builtin_fmaxf(most, v[k]);
      }
      most = wave_max(most);
      referred = most > kNothing;
      const float t = __builtin_fmaxf((before.m - most) * kLog2E, kNoPower), c = __builtin_amdgcn_exp2f(t);
      sums = {most, c * before.s, ENTROPY ? c * __builtin_fmaf(t, before.s, before.w) : 0.f};
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (first(j) >= v1) break;
        float v[8];
        get(j, v);
        add(v);
      }
    }
  }
  if (__any(!(sums.s + sums.w < __builtin_inff())) || !referred) {
    auto each = [&](auto f) {
#pragma unroll 2
      for (int at = v0 + thread * 8; at < v1; at += 512 * W) {
        const int begin = !vector || at < a.V - 8 ? at : a.V - 8;
        float v[8];
        if (vector) {
          Eight<AT> q;
          q.load(row + begin);
          q.get(v);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = at + k < v1 ? load_f32(row + at + k) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (begin + k >= at && begin + k < v1) f(v[k]);
      }
    };
    float most = kLowest;
    each([&](float v) { most = __builtin_fmaxf(most, v); });
    sums = {wave_max(most), 0.f, 0.f};
    each([&](float v) {
      const float t = __builtin_elementwise_maximum((v - sums.m) * kLog2E, kNoPower), e = __builtin_amdgcn_exp2f(t);
      sums.s += e;
      sums.w = __builtin_fmaf(t, e, sums.w);
    });
  }
  sums.s = wave_sum(sums.s);
  if (ENTROPY) sums.w = wave_sum(sums.w);
  if constexpr (W > 1) {
    if (lane == 0) sums_of[wave][0] = sums.m, sums_of[wave][1] = sums.s, sums_of[wave][2] = sums.w;
    __syncthreads();
    if (wave > 0) return;
    sums = lane < W ? RowSums{sums_of[lane % W][0], sums_of[lane % W][1], sums_of[lane % W][2]} : RowSums{kLowest, 0.f, 0.f};
    sums = join_sums(sums);
  }
  if (thread > 0) return;
  if (a.splits > 1) {
    float* part = a.part + (r * a.splits + split) * 4;
    part[0] = sums.m, part[1] = sums.s, part[2] = sums.w;
  } else {
    row_results<AT>(a, r, target, sums);
  }
}

// The pieces of a row joined.  One workgroup per row.  The alternatives of the pieces are sorted lists: with P of them, the least of their ceil(top_k / P)-th
// ones is reached by top_k at least; what reaches it finds its rank among what does.  One row of 131072 with 20 alternatives, 16 pieces:
// 3.4 us of 8.6 (by itself; with a rank among all 320 of them 5.8).
constexpr int kJoinInLds = 4096;
template <typename AT>
__global__ __launch_bounds__(1024) void k_token_scores_join(ScoresArgs a) {
  __shared__ unsigned long long list[kJoinInLds];
  __shared__ int listed;
  const int threads = blockDim.x;
  const long long r = blockIdx.x;
  const long long target = a.targets ? a.targets[r] : 0;
  if (target < 0) {
    no_row(a, r, threadIdx.x, threads);
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
  unsigned bound = 0xFFFFFFFFu;
  for (int p = lane; p < a.splits; p += 64) {
    const unsigned reach = (unsigned)(all[(long long)p * a.top_k + (a.top_k - 1) / a.splits] >> 32);
    bound = reach < bound ? reach : bound;
  }
  bound = wave_min(bound);
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  for (long long j = threadIdx.x; j < n; j += threads) {
    const unsigned long long q = all[j];
    if ((unsigned)(q >> 32) >= bound) {
      const int at = atomicAdd(&listed, 1);
      if (at < kJoinInLds) list[at] = q;
    }
  }
  __syncthreads();
  auto put = [&](int rank, unsigned long long q) {
    if ((lane & 15) == 0 && rank < a.top_k) {
      a.top_log_prob[r * a.top_k + rank] = norm.log_prob(logit_of(q));
      a.top_ids[r * a.top_k + rank] = (int64_t)(unsigned)~(unsigned)q;
    }
  };
  if (listed <= kJoinInLds) {
    const int count = listed;
    for (int j = threadIdx.x >> 4; j < count; j += threads >> 4) {
      const unsigned long long q = list[j];
      put(rank_in(list, count, q, lane), q);
    }
    return;
  }
  // Too many (there are more than 64 pieces, of logits most of which are equal): 16 lanes look at 16 of the pieces' lists at once, by halving.
  for (long long j = threadIdx.x >> 4; j < n; j += threads >> 4) {
    const unsigned long long q = all[j];
    int rank = 0;
    for (int p0 = 0; p0 < a.splits && rank < a.top_k; p0 += 16) {
      const int p = p0 + (lane & 15);
      int low = 0, high = p < a.splits ? a.top_k : 0;  // how many of piece p are larger
      while (low < high) {
        const int mid = (low + high) / 2;
        if (all[(long long)p * a.top_k + mid] > q)
          low = mid + 1;
        else
          high = mid;
      }
      rank += quarter_sum(low);
    }
    put(rank, q);
  }
}

// D = p (A + B t), plus d_log_prob at the target; t = log2 p / 2.  THREADS: 16 or 64 lanes per row, or 256 for a piece of
// kBwdPiece logits of a row.  The last rows go first: their logits, which the forward pass read last, may still lie in the Infinity Cache (4096 rows of 32000
// bf16, a quarter of them without a token, with the forward pass: 141 us from the first row on, 137 from the last, 122 with results stored past the caches
// as well).  Bound by memory: 70 us of those, 459 MB.
constexpr int kBwdPiece = 8192;
template <typename AT, int THREADS>
__global__ __launch_bounds__(256) void k_token_scores_bwd(ScoresArgs a) {
  constexpr bool ROW = THREADS < 256;
  constexpr int N = ROW ? 1 : kBwdPiece / (256 * 8);
  const int thread = threadIdx.x % THREADS;
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const long long item = ROW ? block * (256ll / THREADS) + threadIdx.x / THREADS : block;
  if (ROW && item >= a.rows) return;
  const long long r = ROW ? item : (unsigned)item / (unsigned)a.splits, v0 = ROW ? 0 : (item - r * a.splits) * kBwdPiece;
  const long long v1 = ROW ? a.V : (v0 + kBwdPiece < a.V ? v0 + kBwdPiece : a.V);
  const AT* x = (const AT*)a.logits + r * a.ld;
  AT* D = (AT*)a.D + r * a.V;
  const long long target = a.targets ? a.targets[r] : 0;
  const float base = a.norm[2 * r], log_s = a.norm[2 * r + 1];
  const float g = a.d_log_prob ? a.d_log_prob[r] : 0.f, ge = a.d_entropy ? a.d_entropy[r] : 0.f, h = a.d_entropy ? a.entropy[r] : 0.f;
  const bool none = target < 0 || log_s == -__builtin_inff();
  // (The square root of p, twice: p may be below the normal numbers where its products are not.  t is half of log2 p.)
  const float A = a.targets && target >= a.V ? __builtin_nanf("") : -__builtin_fmaf(ge, h, g), B = -2.f * kLn2 * ge, c = -0.5f * kLog2E * log_s;
  auto one = [&](float v) {
    const float t = __builtin_elementwise_maximum(__builtin_fmaf(v - base, 0.5f * kLog2E, c), kNoPower), root = __builtin_amdgcn_exp2f(t);
    return root * (root * __builtin_fmaf(B, t, A));
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
        q[j].store_streamed(D + at);
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
