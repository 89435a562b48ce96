// gfx950 kernel of dropout from a counter: the mask is computed where it is applied, forward and backward, and never stored.
#pragma once

#include "sequence_common.h"

namespace rtn {

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  long long ldx, ldr;
  long long times, rows, width;  // of x; without a mask for all frames, all rows are of one time
  long long count;  // elements of the mask
  long long frames;               // that share a mask and are dealt to one thread
  unsigned threshold;
  float scale;
  unsigned key0, key1;
  unsigned long long offset;
  const int64_t* offset_ptr;
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

// Scale or drop the eight elements of a group, and add.
template <typename AT, bool ADD>
__device__ __forceinline__ void drop(Eight<AT>& x, const Eight<AT>& r, const Draws& draws, unsigned threshold, float scale) {
  float v[8], add[8];
  x.get(v);
  if (ADD) r.get(add);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] = draws.of(k) >= threshold ? v[k] * scale : 0.f;  // (not a product with 0: a dropped NaN is gone)
    if (ADD) v[k] += add[k];
  }
  x.set(v);
}

// x, y and residual without gaps: one row of `count` elements, or `times` of them (SHARED).  A thread takes the groups g and g + 256 of
// its workgroup's 512, in SHARED one group for `frames` frames (blockIdx.y: which ones).
template <typename AT, bool ADD, bool SHARED>
__global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
  constexpr int G = SHARED ? 1 : 2;
  const unsigned long long offset = a.offset + (a.offset_ptr ? (unsigned long long)*a.offset_ptr : 0ull);
  const long long g0 = blockIdx.x * (256ll * G) + threadIdx.x;
  if (!SHARED && (g0 + 256 * (G - 1)) * 8 + 8 <= a.count) {
    Eight<AT> x[G], r[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      x[j].load((const AT*)a.x + (g0 + 256 * j) * 8);
      if (ADD) r[j].load((const AT*)a.residual + (g0 + 256 * j) * 8);
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      drop<AT, ADD>(x[j], r[j], philox((unsigned long long)(g0 + 256 * j), offset, a.key0, a.key1), a.threshold, a.scale);
      x[j].store_streamed((AT*)a.y + (g0 + 256 * j) * 8);
    }
    return;
  }
  const long long t0 = SHARED ? blockIdx.y * a.frames : 0, t1 = SHARED ? (t0 + a.frames < a.times ? t0 + a.frames : a.times) : 1;
#pragma unroll 1
  for (int j = 0; j < G; ++j) {
    const long long g = g0 + 256 * j, e = g * 8;
    if (e >= a.count) break;
    const Draws draws = philox((unsigned long long)g, offset, a.key0, a.key1);
    if (e + 8 <= a.count) {
      const AT* x = (const AT*)a.x + t0 * a.count + e;
      const AT* r = (const AT*)a.residual + (ADD ? t0 * a.count + e : 0);
      AT* y = (AT*)a.y + t0 * a.count + e;
#pragma unroll 4
      for (long long t = t0; t < t1; ++t, x += a.count, y += a.count) {
        Eight<AT> v, w;
        v.load(x);
        if (ADD) w.load(r), r += a.count;
        drop<AT, ADD>(v, w, draws, a.threshold, a.scale);
        v.store(y);
      }
    } else {  // the last elements
#pragma unroll 1
      for (long long t = t0; t < t1; ++t)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e + k < a.count) {
            const long long at = t * a.count + e + k;
            float v = draws.of(k) >= a.threshold ? load_f32((const AT*)a.x + at) * a.scale : 0.f;
            if (ADD) v += load_f32((const AT*)a.residual + at);
            store_f32((AT*)a.y + at, v);
          }
    }
  }
}

// Rows with a pitch: one thread per group of the mask, for all frames that share it.
template <typename AT, bool ADD>
__global__ __launch_bounds__(256) void k_dropout_rows(DropoutArgs a) {
  const long long g = blockIdx.x * 256ll + threadIdx.x, e = g * 8;
  if (e >= a.count) return;
  const unsigned long long offset = a.offset + (a.offset_ptr ? (unsigned long long)*a.offset_ptr : 0ull);
  const Draws draws = philox((unsigned long long)g, offset, a.key0, a.key1);
  const long long row0 = a.count >> 32 ? e / a.width : (long long)((unsigned)e / (unsigned)a.width), col = e - row0 * a.width;
#pragma unroll 1
  for (long long t = 0; t < a.times; ++t) {
    long long row = t * a.rows + row0, c = col;
    if (col + 8 <= a.width) {
      Eight<AT> v, w;
      v.load((const AT*)a.x + row * a.ldx + c);
      if (ADD) w.load((const AT*)a.residual + row * a.ldr + c);
      drop<AT, ADD>(v, w, draws, a.threshold, a.scale);
      v.store((AT*)a.y + row * a.width + c);
      continue;
    }
    // the end of a row, and what follows of the next ones
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (e + k >= a.count) break;
      float v = draws.of(k) >= a.threshold ? load_f32((const AT*)a.x + row * a.ldx + c) * a.scale : 0.f;
      if (ADD) v += load_f32((const AT*)a.residual + row * a.ldr + c);
      store_f32((AT*)a.y + row * a.width + c, v);
      if (++c == a.width) c = 0, ++row;
    }
  }
}

}  // namespace rtn
