// What the kernels that rank tokens share: numbers in the order of logits and their indices, and joins over the lanes of a wavefront.
#pragma once

#include <type_traits>

#include "sequence_common.h"

namespace rtn {

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

}  // namespace rtn
