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

// x, y and residual without gaps: one row of `count` elements, or `times` of them with one mask (SHARED), whose groups follow each other from row to row.  A
// thread takes the groups i and i + 256 of its workgroup's 512.  Bound by memory: [1000,32,1024] bf16 with a residual 36 us (196 MB, 5.4 TB/s), without
// 21 over several inputs in turn (131 MB, 6.3; 26.5 with stores that stay in the caches), as the gradient behind such a forward pass 22.6 to 24.5.  The draws of a group are made anew for every frame that shares
// them: with a thread for up to 16 frames of a group 29.1 us instead of 22.7.
template <typename AT, bool ADD, bool SHARED>
__global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
  constexpr int G = 2;
  const unsigned long long offset = a.offset + (a.offset_ptr ? (unsigned long long)*a.offset_ptr : 0ull);
  const long long groups = (a.count + 7) / 8, items = SHARED ? groups * a.times : groups;
  const long long i0 = blockIdx.x * (256ll * G) + threadIdx.x;
  long long group[G], first[G];  // of the mask; the first element in x
  bool whole[G];
  Eight<AT> x[G], r[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const long long i = i0 + 256 * j, t = !SHARED ? 0 : (items >> 32 ? i / groups : (long long)((unsigned)i / (unsigned)groups));
    group[j] = i - t * groups;
    first[j] = t * a.count + group[j] * 8;
    whole[j] = i < items && group[j] * 8 + 8 <= a.count;
    if (whole[j]) {
      x[j].load((const AT*)a.x + first[j]);
      if (ADD) r[j].load((const AT*)a.residual + first[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const Draws draws = philox((unsigned long long)group[j], offset, a.key0, a.key1);
    if (whole[j]) {
      drop<AT, ADD>(x[j], r[j], draws, a.threshold, a.scale);
      x[j].store_streamed((AT*)a.y + first[j]);
    } else if (i0 + 256 * j < items) {  // the last ones of the mask
      const int left = (int)(a.count - group[j] * 8);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) {
          float v = draws.of(k) >= a.threshold ? load_f32((const AT*)a.x + first[j] + k) * a.scale : 0.f;
          if (ADD) v += load_f32((const AT*)a.residual + first[j] + k);
          store_f32((AT*)a.y + first[j] + k, v);
        }
    }
  }
}

// Rows with a pitch: one thread per group of the mask, for every gridDim.y-th of the frames that share it.  [1000,32,500] bf16 in rows of 512: 19 us (64 MB, 3.3 TB/s;
// one group in 63 takes the way of single elements, and nearly every wavefront has one.  Two vectors, of the row's end and of the next one's beginning, would do where
// rows are not shorter than eight).
template <typename AT, bool ADD>
__global__ __launch_bounds__(256) void k_dropout_rows(DropoutArgs a) {
  const long long g = blockIdx.x * 256ll + threadIdx.x, e = g * 8;
  if (e >= a.count) return;
  const unsigned long long offset = a.offset + (a.offset_ptr ? (unsigned long long)*a.offset_ptr : 0ull);
  const Draws draws = philox((unsigned long long)g, offset, a.key0, a.key1);
  const long long row0 = a.count >> 32 ? e / a.width : (long long)((unsigned)e / (unsigned)a.width), col = e - row0 * a.width;
#pragma unroll 1
  for (long long t = blockIdx.y; t < a.times; t += gridDim.y) {
    long long row = t * a.rows + row0, c = col;
    if (col + 8 <= a.width) {
      Eight<AT> v, w;
      v.load((const AT*)a.x + row * a.ldx + c);
      if (ADD) w.load((const AT*)a.residual + row * a.ldr + c);
      drop<AT, ADD>(v, w, draws, a.threshold, a.scale);
      v.store((AT*)a.y + row * a.width + c);
      continue;
    }
    // the end of a row, and what follows of the next ones: all of it is loaded before any of it is stored
    float v[8], add[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (e + k >= a.count) break;
      v[k] = load_f32((const AT*)a.x + row * a.ldx + c);
      if (ADD) add[k] = load_f32((const AT*)a.residual + row * a.ldr + c);
      if (++c == a.width) c = 0, ++row;
    }
    AT* y = (AT*)a.y + (t * a.rows + row0) * a.width + col;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (e + k >= a.count) break;
      v[k] = draws.of(k) >= a.threshold ? v[k] * a.scale : 0.f;
      if (ADD) v[k] += add[k];
      store_f32(y + k, v[k]);
    }
  }
}

}  // namespace rtn
