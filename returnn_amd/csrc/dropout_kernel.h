// gfx950 kernel of dropout from a counter: the mask is computed where it is applied, forward and backward, and never stored.
#pragma once

#include "sequence_common.h"

namespace rtn {

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  long long ldx, ldr;
  long long times, rows, width;
  unsigned threshold;
  float scale;
  unsigned key0, key1;
  unsigned long long offset;
  const int64_t* offset_ptr;
  int same_over_time;
};

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, 2011).
struct Draws {
  unsigned w[4];
  // the 16-bit draw of element k = 0..7 of the group
  __device__ __forceinline__ unsigned of(int k) const { return k & 1 ? w[k >> 1] >> 16 : w[k >> 1] & 0xFFFFu; }
};
__device__ __forceinline__ Draws philox(unsigned long long group, unsigned long long offset, unsigned key0, unsigned key1) {
  unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32), c2 = (unsigned)offset, c3 = (unsigned)(offset >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long p0 = (unsigned long long)c0 * 0xD2511F53u, p1 = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(p1 >> 32) ^ c1 ^ key0;
    c2 = (unsigned)(p0 >> 32) ^ c3 ^ key1;
    c1 = (unsigned)p1;
    c3 = (unsigned)p0;
    key0 += 0x9E3779B9u;
    key1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// One thread per group of 8 elements of the mask, over all frames that share it.
template <typename AT>
__global__ void k_dropout(DropoutArgs a) {
  const long long count = (a.same_over_time ? 1 : a.times) * a.rows * a.width, g = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (g * 8 >= count) return;
  const unsigned long long offset = a.offset + (a.offset_ptr ? (unsigned long long)*a.offset_ptr : 0ull);
  const Draws draws = philox((unsigned long long)g, offset, a.key0, a.key1);
  for (long long t = 0; t < (a.same_over_time ? a.times : 1); ++t)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long e = g * 8 + k;
      if (e >= count) break;
      const long long row = e / a.width + t * a.rows, col = e % a.width;
      float v = draws.of(k) >= a.threshold ? load_f32((const AT*)a.x + row * a.ldx + col) * a.scale : 0.f;
      if (a.residual) v += load_f32((const AT*)a.residual + row * a.ldr + col);
      store_f32((AT*)a.y + row * a.width + col, v);
    }
}

}  // namespace rtn
