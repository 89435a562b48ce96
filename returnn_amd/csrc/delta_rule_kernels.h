// gfx950 kernels of the gated delta rule: a recurrence whose state is a matrix per head.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = b_t (v_t - a_t S_{t-1}^T k_t),   o_t = s S_t^T q_t,   a_t = e^{g_t}
#pragma once

#include <type_traits>

#include "sequence_common.h"

namespace rtn {

struct DeltaArgs {
  const void *q, *k, *v;
  long long ldq, ldk, ldv;  // elements from one frame's row to the next
  const float *g, *beta;    // [T,B,H]
  const float* s0;
  const int64_t* lens;
  void* y;
  float* sN;
  long long T;
  int B, key_heads, heads, dk, dv;
  float scale;
  int reverse;
};

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float delta_f32x4;
typedef delta_f32x4 __attribute__((aligned(4))) delta_f32x4_any;

// Frame by frame: 64 columns of a head's state per workgroup, each thread 4 columns of R of the 16 R rows in registers.  What a state gives to a key and to a query is one
// pass over it: S_t^T q = a S_{t-1}^T q + (k.q) u.  A single frame is bound by a launch and the state's way in and out (12 sequences of 8 heads of 128 x 128: 5.9 us for 12.6 MB; 64: 11.7, 5.7 TB/s; 7.1 and
// 14.3 where a row was loaded on a lane's condition);
// further ones by the sums' way through shuffles and LDS, 1.3 us each (2.2 where a frame's numbers were asked for when they were needed).
template <typename AT, int R>
__global__ __launch_bounds__(256) void k_delta_steps(DeltaArgs a) {
  __shared__ float parts[2][4][16][9];
  const int strips = (a.dv + 63) / 64, strip = blockIdx.x % strips, bh = blockIdx.x / strips, b = bh / a.heads, h = bh - b * a.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = strip * 64 + (lane & 15) * 4, row = (wave * 4 + (lane >> 4)) * R;
  const int kh = h / (a.heads / a.key_heads);
  const long long n = frames_of(a.lens, b, a.T);
  const long long matrix = ((long long)b * a.heads + h) * a.dk * a.dv;
  const bool whole = col + 4 <= a.dv;
  // A frame's numbers, asked for a frame ahead.  (What is not there is read at the end of what is, and taken as 0: what is loaded on a condition of a lane is waited for at once.)
  struct Frame {
    AT k[R], q[R], v[4];
    float g, beta;
    long long at;
  } next;
  auto load = [&](long long p) {
    const long long frame = (a.reverse ? n - 1 - p : p) * a.B + b;
    const AT *kp = (const AT*)a.k + frame * a.ldk + kh * a.dk, *qp = (const AT*)a.q + frame * a.ldq + kh * a.dk, *vp = (const AT*)a.v + frame * a.ldv + h * a.dv;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = row + i < a.dk ? row + i : a.dk - 1;
      next.k[i] = kp[e], next.q[i] = qp[e];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) next.v[c] = vp[col + c < a.dv ? col + c : a.dv - 1];
    next.g = a.g[frame * a.heads + h], next.beta = a.beta[frame * a.heads + h], next.at = frame;
  };
  if (n) load(0);
  float S[R][4] = {};
  if (a.s0 && a.dv % 4 == 0) {
    delta_f32x4 w[R];
#pragma unroll
    for (int i = 0; i < R; ++i) w[i] = *(const delta_f32x4_any*)(a.s0 + (matrix + (long long)(row + i < a.dk ? row + i : a.dk - 1) * a.dv + (whole ? col : 0)));
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = row + i < a.dk ? w[i][c] : 0.f;
  } else if (a.s0) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = row + i < a.dk && col + c < a.dv ? a.s0[matrix + (long long)(row + i) * a.dv + col + c] : 0.f;
  }
  for (long long p = 0; p < n; ++p) {
    float k[R], q[R], v[4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool in = row + i < a.dk;
      k[i] = in ? (float)next.k[i] : 0.f;
      q[i] = in ? (float)next.q[i] : 0.f;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = (float)next.v[c];
    const float decay = expf(next.g), beta = next.beta;
    const long long frame = next.at;
    load(p + 1 < n ? p + 1 : p);
    float sum[9] = {};
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        sum[c] = __builtin_fmaf(S[i][c], k[i], sum[c]);
        sum[4 + c] = __builtin_fmaf(S[i][c], q[i], sum[4 + c]);
      }
      sum[8] = __builtin_fmaf(k[i], q[i], sum[8]);
    }
    float(*mine)[16][9] = parts[p & 1];  // (the other one is still being read)
#pragma unroll
    for (int j = 0; j < 9; ++j) {
      sum[j] += __shfl_xor(sum[j], 16);
      sum[j] += __shfl_xor(sum[j], 32);
    }
    if (lane < 16)
#pragma unroll
      for (int j = 0; j < 9; ++j) mine[wave][lane][j] = sum[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 9; ++j) sum[j] = (mine[0][lane & 15][j] + mine[1][lane & 15][j]) + (mine[2][lane & 15][j] + mine[3][lane & 15][j]);
    AT* yp = (AT*)a.y + (frame * a.heads + h) * a.dv;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float u = beta * (v[c] - decay * sum[c]);
      if (row == 0 && col + c < a.dv) store_f32(yp + col + c, a.scale * __builtin_fmaf(decay, sum[4 + c], sum[8] * u));
#pragma unroll
      for (int i = 0; i < R; ++i) S[i][c] = __builtin_fmaf(decay, S[i][c], k[i] * u);
    }
  }
  if (row == 0)
    for (long long t = n; t < a.T; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (col + c < a.dv) store_f32((AT*)a.y + ((t * a.B + b) * a.heads + h) * a.dv + col + c, 0.f);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (row + i < a.dk) {
      const long long at = matrix + (long long)(row + i) * a.dv + col;
      if (whole)
        *(delta_f32x4_any*)(a.sN + at) = (delta_f32x4){S[i][0], S[i][1], S[i][2], S[i][3]};
      else
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (col + c < a.dv) a.sN[at + c] = S[i][c];
    }
}

// ---- in chunks --------------------------------------------------------------------------------------------------------
//
// C frames at once.  With G_i the sum of g up to frame i of the chunk, c_i = e^{G_i}, gamma_i = e^{G_C - G_i}, E_ij = e^{G_i - G_j} (i >= j, so that no power is above 1),
// L_ij = E_ij k_i.k_j (i > j), P_ij = E_ij q_i.k_j (i >= j), T = (1 + diag(beta) L)^-1 and S the state before the chunk:
//
//   U = T diag(beta) (V - diag(c) K S),   Y = scale (diag(c) Q S + P U),   S' = c_C S + K^T diag(gamma) U
//
// k_delta_chunks leaves T, P, L and the powers of every chunk, all chunks side by side; k_delta_forward goes through the chunks of a head.
//
// Matrix instructions take bfloat16 and add in float32.  A float32 number goes in as up to three bfloat16 whose sum it is (8 bits of it each), a product of two of them as
// those products of parts that count: with all whose order is below 3, 2^-24 of it is lost.  So too where the result is rounded to bfloat16 in the end: what it is the sum of (S and U, of which a write may take
// away what the state holds) can be a thousand times as large, and with two parts 2^-17 of that would be lost.
//
// Where a matrix of 32 rows comes out of 16 x 16 tiles and goes into the next product as its right operand, nothing is moved: lane (quarter q, i) has column i
// and, of tile t, rows 4 q + r; the operand wants rows 8 q + 0..7 of it.  So tile t is made of rows 8 q + 4 t + r, which its left operand's lane i = 4 q + r reads.  Left operands lie in LDS
// with rows in that order (position 16 t + 4 q + r), so that a tile's are neighbours.
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 delta_bf16x8;
typedef __attribute__((__vector_size__(8 * sizeof(float)))) float delta_f32x8;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short delta_s16x4;

template <typename AT>
struct DeltaChunk;
template <>
struct DeltaChunk<__bf16> {
  static constexpr int kFrames = 64, kInput = 1;  // frames; parts of an input
};
template <>
struct DeltaChunk<float> {
  static constexpr int kFrames = 32, kInput = 3;  // (K and Q in three parts: 32 frames are what fits into LDS)
};
constexpr int delta_blocks(int frames) { return frames == 64 ? 3 : 1; }  // of 32 x 32, of a lower triangular matrix
// What is kept of a chunk, in numbers of float32: T and P in three parts each, as they lie in LDS (DeltaTile, blocks (0,0), (1,0), (1,1)); L, block by block, row-major; c, gamma, beta,
// and G in two parts.
constexpr int delta_image(int frames) { return 6 * delta_blocks(frames) * 1024 / 2; }
constexpr int delta_record(int frames) { return delta_image(frames) + delta_blocks(frames) * 1024 + 5 * frames; }

struct DeltaChunkArgs {
  DeltaArgs f;
  int chunks;      // of T frames
  float* records;  // [B,heads,chunks][record]
  float* states;   // [B,heads,chunks][DK][dv] before each chunk (DK: dk as in LDS), or NULL
  float* writes;   // [B,heads,chunks][C][dv]: U, or NULL
  const void* dy;
  long long lddy;
  const float* dsN;
  float *dstates, *dwrites;  // as states (behind each chunk) and writes (of diag(beta)'s right side), of the gradient
  void *dq, *dk, *dv;
  float *dq_each, *dk_each;  // [T,B,heads,dk], where heads share queries and keys
  float *dg, *dbeta, *ds0;
  int segments, per;  // of a sequence's chunks, and chunks of each
  float* borders;     // [B,heads,segments - 1][DK][dv]: the state between two segments, or its error
  // [B,heads,segments - 1][3][DK][DK]: what a segment makes of the state before it, in three parts, as a left operand; and transposed
  __bf16 *through, *through_t;
};

__device__ __forceinline__ int delta_place(int row) { return (row & ~31) | ((row >> 2 & 1) << 4) | ((row >> 3 & 3) << 2) | (row & 3); }

// Where an element of a DK x DK matrix lies that is kept as left operands: tile by tile of 16 places and 32 columns, lane by lane, so that a wavefront's read of one is 1 KB.
template <int DK>
__device__ __forceinline__ int delta_left_at(int row, int col) {
  const int place = delta_place(row);
  return (((place >> 4) * (DK / 32) + (col >> 5)) * 64 + (col >> 3 & 3) * 16 + (place & 15)) * 8 + (col & 7);
}

// Eight numbers as N parts, by pairs (element by element the compiler rounds each of them twice).
template <int N>
__device__ __forceinline__ void delta_parts(delta_f32x8 x, delta_bf16x8 (&p)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    seq_u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = pack_bf16(x[2 * k], x[2 * k + 1]);
      if (n + 1 < N) {
        x[2 * k] -= __builtin_bit_cast(float, (unsigned)w[k] << 16);
        x[2 * k + 1] -= __builtin_bit_cast(float, (unsigned)w[k] & 0xFFFF0000u);
      }
    }
    p[n] = __builtin_bit_cast(delta_bf16x8, w);
  }
}
template <int N>
__device__ __forceinline__ void delta_parts(delta_f32x4 a, delta_f32x4 b, delta_bf16x8 (&p)[N]) {
  delta_parts(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), p);
}
// c + a b, the smallest products first.
template <int NA, int NB>
__device__ __forceinline__ delta_f32x4 delta_mma(const delta_bf16x8 (&a)[NA], const delta_bf16x8 (&b)[NB], delta_f32x4 c) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      if (i < NA && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
  return c;
}

// The same for several tiles with one right operand, tile after tile, so that no product waits for the one before it.
template <int TILES, int NA, int NB>
__device__ __forceinline__ void delta_mma(const delta_bf16x8 (&a)[TILES][NA], const delta_bf16x8 (&b)[NB], delta_f32x4* c) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      if (i < NA && s - i < NB) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) c[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[t][i], b[s - i], c[t], 0, 0, 0);
      }
}
// Between what is asked for and the products that do not need it yet: left to itself the compiler reads every operand just before its product, and each of these waits for LDS.
__device__ __forceinline__ void delta_ahead() { __builtin_amdgcn_sched_barrier(0); }

// A matrix in LDS as N planes of R rows of COLS columns, without gaps.  Groups of eight columns change places by the row, so that 16 neighbouring rows of a column lie in different banks, and
// so do four rows of four neighbouring groups.
template <int N, int R, int COLS>
struct DeltaTile {
  alignas(16) char bytes[N][R * COLS * 2];
  static __device__ __forceinline__ int swap_of(int place) {
    const int low = place & 3, high = place >> 2 & 3;
    return COLS == 128 ? low << 2 | high : (COLS == 64 ? (low >> 1) << 2 | high : high);
  }
  static __device__ __forceinline__ int offset(int place, int col) { return place * (COLS * 2) + (((col >> 3) ^ swap_of(place)) << 4) + (col & 7) * 2; }
  __device__ __forceinline__ void put(int place, int col, const delta_bf16x8 (&p)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) *(delta_bf16x8*)(bytes[n] + offset(place, col)) = p[n];
  }
  // Left operand, 16 rows from `place` on and 32 columns from `col` on.  (Or a right operand, of the transposed matrix.)  FIRST: its first plane.
  template <int FIRST = 0, int M>
  __device__ __forceinline__ void left(int place, int col, delta_bf16x8 (&p)[M]) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < M; ++n) p[n] = *(const delta_bf16x8*)(bytes[FIRST + n] + place * (COLS * 2) + offset(lane & 15, col + (lane >> 4) * 8));
  }
  // Left operand of the transposed matrix: rows are the columns 8 q + 4 t + r of the 32 from `col` on, columns the 32 rows from `place` on.
  template <int FIRST = 0, int M>
  __device__ __forceinline__ void transposed(int place, int col, int t, delta_bf16x8 (&p)[M]) const {
    across<FIRST>(place, col + 4 * t, 8, p);
  }
  // Right operand: the 32 rows from `place` on, the 16 columns from `col` on.
  template <int M>
  __device__ __forceinline__ void right(int place, int col, delta_bf16x8 (&p)[M]) const {
    across<0>(place, col, 4, p);
  }
  // What a lane has of a result in rows place + 4 q + r, columns col + i: four rows of it.
  __device__ __forceinline__ delta_f32x4 of_result(int place, int col) const {
    delta_f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = N - 1; n >= 0; --n) {
      const delta_s16x4 v = four(n, place, col, 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] += __builtin_bit_cast(float, (unsigned)(unsigned short)v[r] << 16);
    }
    return x;
  }

 private:
  // The hardware's transposed read: of 16 lanes, lane 4 r + c gives the address of four neighbours in row r, and lane i gets number i % 4 of lane 4 r + i / 4's for r = 0..3.
  __device__ __forceinline__ delta_s16x4 four(int n, int place, int col, int step) const {
    const int lane = threadIdx.x & 63, i = lane & 15;
    const char* at = bytes[n] + place * (COLS * 2) + offset((lane >> 4) * 4 + (i >> 2), col + step * (i & 3));
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) delta_s16x4*)at);
  }
  template <int FIRST, int M>
  __device__ __forceinline__ void across(int place, int col, int step, delta_bf16x8 (&p)[M]) const {
#pragma unroll
    for (int n = 0; n < M; ++n) {
      const delta_s16x4 a = four(FIRST + n, place, col, step), b = four(FIRST + n, place + 16, col, step);
      p[n] = __builtin_bit_cast(delta_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Eight neighbours of a row, of which it has `left`, and 0 behind them.
__device__ __forceinline__ int delta_left(int col, int width) { return width - col < 0 ? 0 : (width - col < 8 ? width - col : 8); }
__device__ __forceinline__ delta_f32x8 delta_load8(const float* at, int left) {
  if (left == 8) {
    const delta_f32x4 a = *(const delta_f32x4_any*)at, b = *(const delta_f32x4_any*)(at + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  delta_f32x8 x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = j < left ? at[j] : 0.f;
  return x;
}
__device__ __forceinline__ delta_bf16x8 delta_load8(const __bf16* at, int left) {
  if (left == 8) return __builtin_bit_cast(delta_bf16x8, *(const seq_u32x4_any*)at);
  delta_bf16x8 x;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = j < left ? at[j] : (__bf16)0.f;
  return x;
}
// The same without a condition of a lane, so that no load is waited for early: the last eight of a row are read in place of what goes beyond its end (of a narrow row its elements one by
// one, the last one for what there is not), and moved to where they belong later, by delta_placed.
__device__ __forceinline__ int delta_read_col(int col, int width) { return width >= 8 ? (col < width - 8 ? col : width - 8) : 0; }
template <bool NARROW = true, typename T>
__device__ __forceinline__ auto delta_load8_any(const T* at, int col, int width) {  // at: column delta_read_col; NARROW: whether there can be fewer than eight
  auto x = delta_load8(at, !NARROW || width >= 8 ? 8 : 0);
  if (NARROW && width < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = at[col + j < width ? col + j : width - 1];
  }
  return x;
}
template <bool NARROW = true, typename E>
__device__ __forceinline__ E delta_placed(E x, int col, int width, bool in) {
  const int shift = width >= 8 ? col - delta_read_col(col, width) : 0;
#pragma unroll
  for (int s = 4; s; s /= 2)
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = shift & s ? (j + s < 8 ? x[j + s] : 0) : x[j];
  if (NARROW && width < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = col + j < width ? x[j] : 0;
  }
  in = in && shift < 8;
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = in ? x[j] : 0;
  return x;
}
__device__ __forceinline__ void delta_parts(delta_bf16x8 x, delta_bf16x8 (&p)[1]) { p[0] = x; }
__device__ __forceinline__ delta_f32x8 delta_wide(delta_f32x8 x) { return x; }
__device__ __forceinline__ delta_f32x8 delta_wide(delta_bf16x8 x) { return __builtin_convertvector(x, delta_f32x8); }

// Which chunk of which head, and where its frames lie: the same in all lanes, and said so, so that addresses are made of scalars.
__device__ __forceinline__ long long delta_same(long long v) {
  return (long long)(unsigned)__builtin_amdgcn_readfirstlane((int)v) | (long long)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}
struct DeltaWhere {
  int b, h, kh, chunk;
  long long n;      // frames of the sequence
  int count;        // of the chunk's frames that it has
  long long first, step;  // row of the chunk's first frame, and from one frame's to the next's
  __device__ __forceinline__ DeltaWhere(const DeltaArgs& a, int bh, int chunk_, int frames) {
    b = bh / a.heads, h = bh - b * a.heads, kh = h / (a.heads / a.key_heads);
    n = delta_same(frames_of(a.lens, b, a.T));
    step = a.reverse ? -(long long)a.B : a.B;
    to(a, chunk_, frames);
  }
  __device__ __forceinline__ void to(const DeltaArgs& a, int chunk_, int frames) {
    chunk = chunk_;
    const long long p = (long long)chunk * frames, left = n - p;
    count = left < 0 ? 0 : (left < frames ? (int)left : frames);
    first = (a.reverse ? n - 1 - p : p) * a.B + b;
  }
  __device__ __forceinline__ long long row(int i) const { return first + i * step; }
};
// The frames of a chunk in a tensor.  Frame i's row of a head, from element `col` on, is at(i) + lane(0, col), or at(0) + lane(i, col) for i up to REACH: at() is made of scalars, lane()
// is an offset of 32 bits (frames are at most kDeltaFrameBytes long) that is the same for all chunks.
constexpr long long kDeltaFrameBytes = 1 << 26;
template <typename T, int REACH>
struct DeltaFrames {
  char* base;
  long long pitch;
  unsigned apart;
  bool turned;
  __device__ __forceinline__ DeltaFrames(const DeltaArgs& a, T* tensor, const DeltaWhere& at, long long ld, long long head)
      : base((char*)(tensor + (at.first * ld + head))), pitch(at.step * ld * (long long)sizeof(T)), apart((unsigned)(a.B * ld * (long long)sizeof(T))), turned(a.reverse) {
    asm("" : "+s"(pitch));  // (its multiples are computed where they are used: kept from chunk to chunk they do not fit into the scalar registers)
    if (turned) base += REACH * pitch;
  }
  __device__ __forceinline__ char* at(int i) const { return base + i * pitch; }
  __device__ __forceinline__ unsigned lane(int i, int col) const { return (unsigned)(turned ? REACH - i : i) * apart + (unsigned)col * (unsigned)sizeof(T); }
};

// Which line and which of its strips a workgroup has.  Neighbouring workgroups go to the eight XCDs in turn; strips of a line, which read the same, are eight apart, on one XCD with its L2.
__device__ __forceinline__ void delta_spread(int strips, int* line, int* strip) {
  const int all = gridDim.x / strips, even = all & ~7, block = blockIdx.x;
  if (block < even * strips) {
    const int eight = block >> 3;
    *strip = eight % strips, *line = eight / strips * 8 + (block & 7);
  } else {
    const int rest = block - even * strips;
    *line = even + rest / strips, *strip = rest % strips;
  }
}

// T, P, L and the powers of a chunk, one workgroup of C / 16 wavefronts each, which have 16 rows of L and P each.  The inverse: diagonal blocks of 16 row by row, a column per
// lane; then T_21 = - T_22 A_21 T_11 for blocks of 16 and of 32, in float32 matrix instructions.  Bound by latency, of rows of K and of 16 steps of a column each, three workgroups on a compute unit: T=1000,
// 32 ragged sequences of 8 heads, keys of 128 in bf16: 88-92 us, 3.1 TB/s, of which the records are the larger part.  (Rows read without a condition, a tile ahead, cost more in selections than they save: 121.)
template <typename AT, int DK>
__global__ __launch_bounds__(DeltaChunk<AT>::kFrames * 4) void k_delta_chunks(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, W = C / 16, BLOCKS = delta_blocks(C), ROW = C + 4;
  __shared__ alignas(16) float A[C * ROW], X[C * ROW], Y[C * ROW];
  __shared__ float high[C], low[C], beta_of[C];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4, i16 = lane & 15;
  const int chunk = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks;
  const DeltaWhere at(a.f, bh, chunk, C);
  // (frames past the end)
  const long long past = a.f.T - (long long)chunk * C;
  for (int i = at.count + wave; i < C && i < past; i += W) {
    AT* y = (AT*)a.f.y + (((long long)chunk * C + i) * a.f.B + at.b) * a.f.heads * a.f.dv + (long long)at.h * a.f.dv;
    for (int e = lane; e < a.f.dv; e += 64) store_f32(y + e, 0.f);
  }
  if (at.count == 0) return;
  float* record = a.records + ((long long)bh * a.chunks + chunk) * delta_record(C);
  float *rL = record + delta_image(C), *rc = rL + BLOCKS * 1024;
  // T (which = 0) or P (1) out of LDS, in three parts, by threads `from` to `to`, eight numbers each.
  auto put_image = [&](int which, const float* of, int from, int to) {
    typedef DeltaTile<6, BLOCKS * 32, 32> Image;
    for (int item = (int)threadIdx.x - from; item >= 0 && item < BLOCKS * 128; item += to - from) {
      const int block = item >> 7, row = item >> 2 & 31, col = (item & 3) * 8;
      const float* x = of + (row + (block > 0) * 32) * ROW + col + (block > 1) * 32;
      delta_bf16x8 parts[3];
      delta_parts(*(const delta_f32x4*)x, *(const delta_f32x4*)(x + 4), parts);
#pragma unroll
      for (int n = 0; n < 3; ++n) *(delta_bf16x8*)((char*)record + (which * 3 + n) * (int)sizeof(Image().bytes[0]) + Image::offset(delta_place(block * 32 + row), col)) = parts[n];
    }
  };
  if (wave == 0) {
    const bool in = lane < at.count;
    const long long f = at.row(in ? lane : 0) * a.f.heads + at.h;
    float g = in ? a.f.g[f] : 0.f;
    const float beta = in ? a.f.beta[f] : 0.f;
    if (g < -200.f) g = -200.f;  // (e^-200 is 0 in float32; sums of minus infinity would give NaN as their difference)
    double G = g;
#pragma unroll
    for (int d = 1; d < C; d *= 2) {
      const double o = __shfl_up(G, d);
      if (lane >= d) G += o;
    }
    const double end = __shfl(G, C - 1);
    if (lane < C) {
      high[lane] = (float)G, low[lane] = (float)(G - (double)(float)G), beta_of[lane] = beta;
      rc[lane] = expf((float)G), rc[C + lane] = expf((float)(end - G)), rc[2 * C + lane] = beta, rc[3 * C + lane] = (float)G, rc[4 * C + lane] = (float)(G - (double)(float)G);
    }
  }
  // 16 rows of K and Q against all up to them
  delta_bf16x8 kf[DK / 32][NI], qf[DK / 32][NI];
  auto fetch = [&](const void* tensor, long long ld, int row, delta_bf16x8(&p)[DK / 32][NI]) {
    const AT* r = (const AT*)tensor + (at.row(row < at.count ? row : 0) * ld + at.kh * a.f.dk + q4 * 8);
#pragma unroll
    for (int b = 0; b < DK / 32; ++b) delta_parts(delta_load8(r + b * 32, row < at.count ? delta_left(b * 32 + q4 * 8, a.f.dk) : 0), p[b]);
  };
  fetch(a.f.k, a.f.ldk, wave * 16 + i16, kf);
  fetch(a.f.q, a.f.ldq, wave * 16 + i16, qf);
  __syncthreads();
  for (int nt = 0; nt < W; ++nt) {
    delta_f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;
    if (nt <= wave) {
      delta_bf16x8 other[DK / 32][NI];
      fetch(a.f.k, a.f.ldk, nt * 16 + i16, other);
#pragma unroll
      for (int b = 0; b < DK / 32; ++b) {
        kk = delta_mma(kf[b], other[b], kk);
        qk = delta_mma(qf[b], other[b], qk);
      }
    }
    const int j = nt * 16 + i16, block = wave / 2 + nt / 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = wave * 16 + q4 * 4 + r;
      const float e = i >= j ? expf((high[i] - high[j]) + (low[i] - low[j])) : 0.f;
      const float l = i > j ? kk[r] * e : 0.f, p = i >= j ? qk[r] * e : 0.f;
      A[i * ROW + j] = beta_of[i] * l;
      X[i * ROW + j] = 0.f;
      Y[i * ROW + j] = p;
      if (nt / 2 <= wave / 2) {
        rL[block * 1024 + (i & 31) * 32 + (j & 31)] = l;
      }
    }
  }
  __syncthreads();
  if (wave) put_image(1, Y, 64, C * 4);
  if (wave == 0 && q4 < W) {
    const float* D = A + (q4 * 16) * ROW + q4 * 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == i16 ? 1.f : 0.f;
#pragma unroll
      for (int l = 0; l < i; ++l) v = __builtin_fmaf(-D[i * ROW + l], x[l], v);
      x[i] = v;
      X[(q4 * 16 + i) * ROW + q4 * 16 + i16] = v;
    }
  }
  __syncthreads();
  // tile (mt, nt) of out = sum over l of left's (mt, l) times right's (l, nt), negated where wanted
  auto product = [&](const float* left, const float* right, float* out, int mt, int nt, int l0, int l1, float sign) {
    delta_f32x4 c = {0.f, 0.f, 0.f, 0.f};
    for (int l = l0 * 16; l < l1 * 16; l += 4)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(left[(mt * 16 + i16) * ROW + l + q4], right[(l + q4) * ROW + nt * 16 + i16], c, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) out[(mt * 16 + q4 * 4 + r) * ROW + nt * 16 + i16] = sign * c[r];
  };
  if (wave & 1) product(A, X, Y, wave, wave - 1, wave - 1, wave, 1.f);
  __syncthreads();
  if (wave & 1) product(X, Y, X, wave, wave - 1, wave, wave + 1, -1.f);
  __syncthreads();
  if constexpr (C == 64) {
    const int mt = 2 + (wave >> 1), nt = wave & 1;
    product(A, X, Y, mt, nt, 0, 2, 1.f);
    __syncthreads();
    product(X, Y, X, mt, nt, 2, 4, -1.f);
    __syncthreads();
  }
  put_image(0, X, 0, C * 4);
}

// What the kernels that go through a head's chunks load of one into LDS, by way of registers: the one behind the next is on its way while one is worked on and the next lies in LDS.
//
// Rows past the end are read as the last one and put as 0.
template <typename AT, int DK, int THREADS, int NP, bool WITH_Q = true>
struct DeltaStage {
  static constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, BLOCKS = delta_blocks(C);
  static constexpr int kApart = THREADS * 8 / DK;  // rows from one of a thread's to the next
  static constexpr int kRows = (C + kApart - 1) / kApart, kImage = ((3 + NP) * BLOCKS * 128 + THREADS - 1) / THREADS, kPowers = (3 * C + THREADS - 1) / THREADS;
  typedef decltype(delta_load8((const AT*)nullptr, 0)) Eight8;
  struct Tiles {
    DeltaTile<NI, C, DK> K;
    DeltaTile<NI, WITH_Q ? C : 1, DK> Q;
    DeltaTile<3 + NP, BLOCKS * 32, 32> TP;  // T, then P
    alignas(16) float powers[3][C];  // c, gamma, beta
  };
  Eight8 k[kRows], q[kRows];
  seq_u32x4 image[kImage];
  float power[kPowers];
  int count;
  // (where threads are more than there is, some do the same)
  static __device__ __forceinline__ int row_of(int n) { return (int)(threadIdx.x / (DK / 8) + n * kApart) % C; }
  static __device__ __forceinline__ int image_of(int n) {
    constexpr int all = (3 + NP) * BLOCKS * 128;
    const int item = n * THREADS + threadIdx.x;
    return all % THREADS == 0 || item < all ? item : all - 1;
  }
  static __device__ __forceinline__ int power_of(int n) {
    const int item = n * THREADS + threadIdx.x;
    return 3 * C % THREADS == 0 || item < 3 * C ? item : 3 * C - 1;
  }
  static __device__ __forceinline__ int place_col() { return threadIdx.x % (DK / 8) * 8; }
  __device__ __forceinline__ void load(const DeltaChunkArgs& a, const DeltaWhere& at, const float* record) {
    count = at.count;
    const DeltaFrames<const AT, C - 1> kf(a.f, (const AT*)a.f.k, at, a.f.ldk, at.kh * a.f.dk), qf(a.f, (const AT*)a.f.q, at, a.f.ldq, at.kh * a.f.dk);
    const int col = delta_read_col(place_col(), a.f.dk);
#pragma unroll
    for (int n = 0; n < kRows; ++n) {
      const int of = row_of(n) < count ? row_of(n) : count - 1;
      k[n] = delta_load8_any<(DK <= 32)>((const AT*)(kf.at(0) + kf.lane(of, col)), place_col(), a.f.dk);
      if constexpr (WITH_Q) q[n] = delta_load8_any<(DK <= 32)>((const AT*)(qf.at(0) + qf.lane(of, col)), place_col(), a.f.dk);
    }
#pragma unroll
    for (int n = 0; n < kImage; ++n) image[n] = *(const seq_u32x4*)((const char*)record + (unsigned)image_of(n) * 16u);
#pragma unroll
    for (int n = 0; n < kPowers; ++n) power[n] = *(const float*)((const char*)(record + delta_image(C) + BLOCKS * 1024) + (unsigned)power_of(n) * 4u);
  }
  __device__ __forceinline__ void store(Tiles& to, int dk) const {
    auto rows = [&](auto whole) {
#pragma unroll
      for (int n = 0; n < kRows; ++n) {
        delta_bf16x8 parts[NI];
        const bool in = decltype(whole)::value || row_of(n) < count;
        delta_parts(decltype(whole)::value ? k[n] : delta_placed<(DK <= 32)>(k[n], place_col(), dk, in), parts);
        to.K.put(delta_place(row_of(n)), place_col(), parts);
        if constexpr (WITH_Q) {
          delta_parts(decltype(whole)::value ? q[n] : delta_placed<(DK <= 32)>(q[n], place_col(), dk, in), parts);
          to.Q.put(delta_place(row_of(n)), place_col(), parts);
        }
      }
    };
    if (count == C && dk == DK)
      rows(std::true_type());
    else
      rows(std::false_type());
#pragma unroll
    for (int n = 0; n < kImage; ++n) *(seq_u32x4*)(&to.TP.bytes[0][0] + image_of(n) * 16) = image[n];
#pragma unroll
    for (int n = 0; n < kPowers; ++n) (&to.powers[0][0])[power_of(n)] = power[n];
  }
};
// Four rows' numbers of tile m.
__device__ __forceinline__ delta_f32x4 delta_rows(const float* of, int m) { return *(const delta_f32x4*)(of + (m >> 1) * 32 + ((threadIdx.x >> 4) & 3) * 8 + (m & 1) * 4); }

// An element on its way, in a register of its own (two of 16 bits in one would be waited for to be joined).
template <typename AT>
struct DeltaElement;
template <>
struct DeltaElement<float> {
  float x;
  __device__ __forceinline__ void load(const void* from) { x = *(const float*)from; }
  __device__ __forceinline__ float get() const { return x; }
};
template <>
struct DeltaElement<__bf16> {
  unsigned x;
  __device__ __forceinline__ void load(const void* from) { x = *(const unsigned short*)from; }
  __device__ __forceinline__ float get() const { return __builtin_bit_cast(float, x << 16); }
};

// Sixteen columns of a head per wavefront, which go through its chunks one after the other, W wavefronts per workgroup, which share what DeltaStage brings: what the forward pass and the
// gradient have alike.  A lane has, of tile m, rows 32 (m / 2) + 8 q + 4 (m % 2) + r.
template <typename AT, int DK, int W>
struct DeltaStrip {
  static constexpr int C = DeltaChunk<AT>::kFrames, M = C / 16, NB = C / 32, KB = DK / 32;
  const DeltaChunkArgs& a;
  int q4, col;
  bool has;
  int strip, bh;
  unsigned lane_state;
  long long pitch_state;  // (bytes)
  int segment;
  // `columns` of all strips; segments from `first` on, as many as there are launched
  __device__ __forceinline__ DeltaStrip(const DeltaChunkArgs& args, int columns, int first, int segments) : a(args) {
    const int lane = threadIdx.x & 63, strips = (columns + 16 * W - 1) / (16 * W);
    q4 = lane >> 4;
    int rest;
    delta_spread(strips, &rest, &strip);
    segment = first + rest % segments, bh = rest / segments;
    col = (strip * W + (int)(threadIdx.x >> 6)) * 16 + (lane & 15);
    has = col < a.f.dv;
    lane_state = (unsigned)(q4 * 8 * a.f.dv + col) * 4u;
    pitch_state = a.f.dv * 4ll;
  }
  __device__ __forceinline__ float* border(int n) const { return a.borders + ((long long)bh * (a.segments - 1) + n) * kept(); }
  static __device__ __forceinline__ constexpr int first_of(int m) { return (m >> 1) * 32 + (m & 1) * 4; }
  __device__ __forceinline__ int row_of(int m, int r) const { return first_of(m) + q4 * 8 + r; }
  __device__ __forceinline__ long long matrix() const { return (long long)a.f.dk * a.f.dv; }
  __device__ __forceinline__ long long kept() const { return (long long)DK * a.f.dv; }
  __device__ __forceinline__ long long number(int chunk) const { return (long long)bh * a.chunks + chunk; }
  // A state, or C rows of float32 of the width dv.
  template <int TILES>
  __device__ __forceinline__ void get(const float* from, int rows, delta_f32x4 (&x)[TILES]) const {
#pragma unroll
    for (int k = 0; k < TILES; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[k][r] = from && has && row_of(k, r) < rows ? *(const float*)((const char*)from + (first_of(k) + r) * pitch_state + lane_state) : 0.f;
  }
  template <int TILES>
  __device__ __forceinline__ void put(float* to, int rows, const delta_f32x4 (&x)[TILES]) const {
    long long pitch = pitch_state;
    asm("" : "+s"(pitch));  // (as of DeltaFrames)
    if (!has) return;
#pragma unroll
    for (int b = 0; b < TILES / 2; ++b) {
      char* row = (char*)to + b * 32 * pitch;
#pragma unroll
      for (int j = 0; j < 8; ++j, row += pitch)
        if (rows == TILES * 16 || b * 32 + q4 * 8 + j < rows) *(float*)(row + lane_state) = x[2 * b + (j >> 2)][j & 3];
    }
  }
  // C frames of a tensor [T,B,heads,dv].  What is no column is computed as the last one, and what is no row is read as the last one and taken as 0.
  __device__ __forceinline__ void load(const void* tensor, long long ld, const DeltaWhere& at, DeltaElement<AT> (&x)[M][4]) const {
    const DeltaFrames<const AT, C - 1> frames(a.f, (const AT*)tensor, at, ld, (long long)at.h * a.f.dv);
    // (one way for whole chunks and others: where ways meet, 16 bits would be waited for to be widened)
    const unsigned step = frames.turned ? 0u - frames.apart : frames.apart;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int last = at.count - 1, first = b * 32 + q4 * 8;
      unsigned lane = frames.lane(first < last ? first : last, has ? col : a.f.dv - 1);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[2 * b + (j >> 2)][j & 3].load(frames.at(0) + lane);
        lane += first + j < last ? step : 0u;
      }
    }
  }
  __device__ __forceinline__ void take(const DeltaElement<AT> (&x)[M][4], int count, delta_f32x4 (&to)[M]) const {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        to[m][r] = x[m][r].get();
        if (count < C) to[m][r] = row_of(m, r) < count ? to[m][r] : 0.f;
      }
  }
  __device__ __forceinline__ void store(void* tensor, const DeltaWhere& at, const delta_f32x4 (&x)[M]) const {
    const DeltaFrames<AT, 24> frames(a.f, (AT*)tensor, at, (long long)a.f.heads * a.f.dv, (long long)at.h * a.f.dv);
    if (!has) return;
    const unsigned lane = frames.lane(q4 * 8, col);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      char* to = frames.at(b * 32);
#pragma unroll
      for (int j = 0; j < 8; ++j, to += frames.pitch)
        if (at.count == C || b * 32 + q4 * 8 + j < at.count) store_f32((AT*)(to + lane), x[2 * b + (j >> 2)][j & 3]);
    }
  }
};
template <int N>
__device__ __forceinline__ void delta_zero(delta_f32x4 (&x)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = (delta_f32x4){0.f, 0.f, 0.f, 0.f};
}

// Where sequences and heads are few, their chunks are dealt to segments that work side by side.  A segment makes B + A S of a state S: a first pass (KIND kDeltaThrough) finds B, the state behind
// it from none before it, and A, its columns from those of the unit matrix without values; k_delta_join goes from segment to segment; then all segments begin with their state.
//
// A chunk needs the one before it, so a workgroup's time is its chain of products, of LDS reads between them and of barriers: 14 us a chunk of 64 frames, keys and values of 128 in bf16, with eight wavefronts
// (matrix instructions 18 %, others 26 %, waiting 50 %).  Hence 16 columns of the state per wavefront, in registers from the first chunk to the last, with U and Y going from product to product without leaving them, and
// everything of the next chunk asked for a chunk ahead.  T=1000, 32 ragged sequences of 8 heads, and all that the gradient wants kept: 225-234 us, 384 MB read, 383 written.  T=4000, one sequence: 30 us for each of
// the two passes.  (Loads on a condition of a lane, each of which the compiler waits for where paths meet again: 300 us for what then took 200.  Outputs
// from three parts of states and writes cost 4 %: one more plane of P, and 15 to 18 registers that go through memory with eight wavefronts and keys of more than 64.)
enum { kDeltaPlain, kDeltaKeep, kDeltaThrough };
template <typename AT, int DK, int W, int KIND>
__global__ __launch_bounds__(64 * W) void k_delta_forward(DeltaChunkArgs a) {
  constexpr bool KEEP = KIND == kDeltaKeep, THROUGH = KIND == kDeltaThrough;
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, M = C / 16, NB = C / 32, KB = DK / 32, BLOCKS = delta_blocks(C);
  typedef DeltaStage<AT, DK, 64 * W, THROUGH ? 0 : 3, !THROUGH> Stage;
  __shared__ typename Stage::Tiles tiles[2];
  const int values = (a.f.dv + 15) / 16 * 16;
  DeltaStrip<AT, DK, W> strip(a, THROUGH ? values + DK : a.f.dv, 0, THROUGH ? a.segments - 1 : a.segments);
  const bool unit = THROUGH && strip.col >= values;  // (the same in all lanes)
  if (THROUGH && strip.segment == 0 && strip.strip * W * 16 >= values) return;
  DeltaWhere at(a.f, strip.bh, 0, C);
  const int all_chunks = (int)((at.n + C - 1) / C), chunk0 = strip.segment * a.per, chunks = all_chunks < chunk0 + a.per ? all_chunks : chunk0 + a.per;
  const float* records = a.records + strip.number(0) * delta_record(C);
  delta_f32x4 S[2 * KB];
  if (THROUGH && strip.segment) {
#pragma unroll
    for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) S[k][r] = strip.row_of(k, r) == strip.col - values ? 1.f : 0.f;
  } else {
    const bool border = strip.segment > 0;
    strip.get(border ? strip.border(strip.segment - 1) : (a.f.s0 ? a.f.s0 + strip.bh * strip.matrix() : nullptr), border ? DK : a.f.dk, S);
  }
  Stage stage;
  DeltaElement<AT> v[M][4];
  auto load = [&](int chunk) {  // (the last one again where there is no next: what is loaded on a condition is waited for)
    at.to(a.f, chunk < chunks ? chunk : chunks - 1, C);
    stage.load(a, at, records + (long long)at.chunk * delta_record(C));
  };
  if (chunk0 < chunks) {
    load(chunk0);
    strip.load(a.f.v, a.f.ldv, at, v);
    stage.store(tiles[chunk0 & 1], a.f.dk);
    load(chunk0 + 1);
    __syncthreads();
  }
  for (int chunk = chunk0; chunk < chunks; ++chunk) {
    const typename Stage::Tiles& lds = tiles[chunk & 1];
    DeltaWhere here = at;
    here.to(a.f, chunk, C);
    delta_f32x4 R[M], O[M], KS[M], U[M];
    strip.take(v, here.count, R);
    strip.load(a.f.v, a.f.ldv, at, v);
    stage.store(tiles[chunk + 1 & 1], a.f.dk);
    load(chunk + 2);
    if (unit) delta_zero(R);
    if (KEEP) strip.put(a.states + strip.number(chunk) * strip.kept(), DK, S);
    delta_zero(KS);
    delta_zero(O);
    delta_zero(U);
    {
      delta_bf16x8 k[2][M][NI], q[2][M][NI], p[2][3];
      auto ask = [&](int b) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          lds.K.left(m * 16, b * 32, k[b & 1][m]);
          if constexpr (!THROUGH) lds.Q.left(m * 16, b * 32, q[b & 1][m]);
        }
      };
      ask(0);
      delta_parts(S[0], S[1], p[0]);
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        if (b + 1 < KB) ask(b + 1);
        delta_ahead();
        if (b + 1 < KB) delta_parts(S[2 * b + 2], S[2 * b + 3], p[b + 1 & 1]);
        delta_mma(k[b & 1], p[b & 1], KS);
        if constexpr (!THROUGH) delta_mma(q[b & 1], p[b & 1], O);
      }
    }
    {
      // T and P: blocks (0,0), (1,0), (1,1), of two tiles of 16 rows each
      delta_bf16x8 t[BLOCKS][2][3], p[BLOCKS][2][3], right[3], some[3];
      auto ask_t = [&](int n) {
        lds.TP.left(n * 32, 0, t[n][0]);
        lds.TP.left(n * 32 + 16, 0, t[n][1]);
      };
      auto ask_p = [&](int n) {
        if constexpr (!THROUGH) {
          lds.TP.template left<3>(n * 32, 0, p[n][0]);
          lds.TP.template left<3>(n * 32 + 16, 0, p[n][1]);
        }
      };
      ask_t(0);
      if constexpr (NB == 2) ask_t(1);
      delta_ahead();
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const delta_f32x4 c = delta_rows(lds.powers[0], m);
        R[m] = delta_rows(lds.powers[2], m) * (R[m] - c * KS[m]);
        O[m] *= c;
      }
      delta_parts(R[0], R[1], right);
      delta_mma(t[0], right, U);
      ask_p(0);
      if constexpr (NB == 2) {
        ask_t(2);
        delta_ahead();
        delta_mma(t[1], right, U + 2);
        delta_parts(R[2], R[3], right);
        delta_parts(U[0], U[1], some);
        delta_mma(t[2], right, U + 2);
        ask_p(1);
        ask_p(2);
        delta_ahead();
        if constexpr (!THROUGH) {
          delta_mma(p[0], some, O);
          delta_mma(p[1], some, O + 2);
          delta_parts(U[2], U[3], some);
          delta_mma(p[2], some, O + 2);
        }
      } else if constexpr (!THROUGH) {
        delta_parts(U[0], U[1], some);
        delta_mma(p[0], some, O);
      }
    }
    if (KEEP) strip.put(a.writes + strip.number(chunk) * C * a.f.dv, C, U);
    {
      delta_bf16x8 k[2][KB][NI], right[NB][3];
      // (half of the tiles at a time)
      auto ask = [&](int n) {
#pragma unroll
        for (int i = 0; i < KB; ++i) lds.K.transposed(n / 2 * 32, (n % 2 * KB + i) / 2 * 32, (n % 2 * KB + i) % 2, k[n & 1][i]);
      };
      ask(0);
      const float end = lds.powers[0][C - 1];
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) S[k] *= end;
#pragma unroll
      for (int b = 0; b < NB; ++b) delta_parts(delta_rows(lds.powers[1], 2 * b) * U[2 * b], delta_rows(lds.powers[1], 2 * b + 1) * U[2 * b + 1], right[b]);
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n) {
        if (n + 1 < 2 * NB) ask(n + 1);
        delta_ahead();
        delta_mma(k[n & 1], right[n / 2], S + n % 2 * KB);
      }
    }
    if constexpr (!THROUGH) {
#pragma unroll
      for (int m = 0; m < M; ++m) O[m] *= a.f.scale;
      strip.store(a.f.y, here, O);
    }
    __syncthreads();
  }
  if constexpr (THROUGH) {
    if (!unit) {
      strip.put(strip.border(strip.segment), DK, S);
    } else if (strip.col < values + DK) {
      const long long first = ((long long)strip.bh * (a.segments - 1) + strip.segment) * 3 * DK * DK;
      const int of = strip.col - values;
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        delta_bf16x8 p[3];
        delta_parts(S[2 * b], S[2 * b + 1], p);
#pragma unroll
        for (int n = 0; n < 3; ++n) {
          if (a.through_t) *(delta_bf16x8*)(a.through_t + first + n * DK * DK + delta_left_at<DK>(of, b * 32 + strip.q4 * 8)) = p[n];
#pragma unroll
          for (int j = 0; j < 8; ++j) a.through[first + n * DK * DK + delta_left_at<DK>(b * 32 + strip.q4 * 8 + j, of)] = p[n][j];
        }
      }
    }
  } else if (strip.segment == (all_chunks ? (all_chunks - 1) / a.per : 0)) {
    strip.put(a.f.sN + strip.bh * strip.matrix(), a.f.dk, S);
  }
}

// States at the segments' borders, one after the other: border n is what segment n (n + 1 for the error of a state, whose segments are gone through from the last one) makes of none, and what it makes
// of the border before it is added.  Sixteen columns per workgroup, 16 rows of them per wavefront; the state goes around through LDS, in parts and as the right operand that all need.
// Bound by what one compute unit gets from memory: 98 KB a border of 128 x 128.  With these read row by row, 64 bytes of each, and asked for a border ahead a border took 2.2 us; in the order of operands,
// 1 KB at a time, three borders ahead, 1.2.
template <typename AT, int DK, bool BACK>
__global__ __launch_bounds__(DK * 4) void k_delta_join(DeltaChunkArgs a) {
  constexpr int KB = DK / 32;
  __shared__ alignas(16) char state[2][KB][3][64][16];
  const int lane = threadIdx.x & 63, k = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, i16 = lane & 15, borders = a.segments - 1;
  int bh, strip;
  delta_spread((a.f.dv + 15) / 16, &bh, &strip);
  const int col = strip * 16 + i16, first = (k >> 1) * 32 + (k & 1) * 4;
  const bool has = col < a.f.dv;
  const long long row = (long long)(first + q4 * 8) * a.f.dv + (has ? col : a.f.dv - 1);
  auto border_of = [&](int n) { return BACK ? borders - 1 - n : n; };
  auto border = [&](int n) { return a.borders + ((long long)bh * borders + border_of(n)) * DK * a.f.dv + row; };
  struct Ahead {  // of a border
    delta_f32x4 own;
    delta_bf16x8 A[KB][3];
  } ahead[3];
  auto get = [&](int n, delta_f32x4& x) {
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = border(n)[r * a.f.dv];
  };
  auto ask = [&](int n, Ahead& of) {
    n = n < borders ? n : borders - 1;
    get(n, of.own);
    const __bf16* from = (BACK ? a.through_t : a.through) + ((long long)bh * borders + border_of(n) + BACK) * 3 * DK * DK;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int m = 0; m < 3; ++m) of.A[b][m] = *(const delta_bf16x8*)(from + m * DK * DK + ((k * KB + b) * 64 + lane) * 8);
  };
  delta_f32x4 S;
  get(0, S);
#pragma unroll
  for (int j = 0; j < 3; ++j) ask(1 + j, ahead[j]);
  auto step = [&](int n, Ahead& now) {
    const delta_f32x4 none = {0.f, 0.f, 0.f, 0.f};
    delta_bf16x8 p[3];
    delta_parts(S, none, p);
#pragma unroll
    for (int m = 0; m < 3; ++m) *(unsigned long long*)(state[n & 1][k >> 1][m][lane] + (k & 1) * 8) = __builtin_bit_cast(seq_u32x4, p[m])[0] | (unsigned long long)__builtin_bit_cast(seq_u32x4, p[m])[1] << 32;
    __syncthreads();
    S = now.own;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
#pragma unroll
      for (int m = 0; m < 3; ++m) p[m] = *(const delta_bf16x8*)state[n & 1][b][m][lane];
      S = delta_mma(now.A[b], p, S);
    }
    if (has)
#pragma unroll
      for (int r = 0; r < 4; ++r) border(n)[r * a.f.dv] = S[r];
    ask(n + 3, now);
  };
  for (int n = 1;; n += 3) {
    step(n, ahead[0]);
    if (n + 1 >= borders) break;
    step(n + 1, ahead[1]);
    if (n + 2 >= borders) break;
    step(n + 2, ahead[2]);
    if (n + 3 >= borders) break;
  }
}

// ---- the gradient -----------------------------------------------------------------------------------------------------
//
// With D the error of the state behind a chunk, S the state before it, U its writes:
//
//   dU = scale P^T dY + diag(gamma) K D,   R = T^T dU,   dV = diag(beta) R,   dS = c_C D + scale Q^T diag(c) dY - K^T diag(beta c) R
//   X = R U^T,  Z = scale dY U^T,  F = Z o E (i >= j),  H = X o diag(beta) E (i > j)
//   dQ = scale diag(c) dY S^T + F K
//   dK = F^T Q + diag(gamma) U D^T - diag(beta c) R S^T - H K - H^T K
//   dbeta_i = R_i.v_i - c_i k_i.(S R_i) - sum_j X_ij L_ij
//   and of G, with N = Z o P - X o diag(beta) L:  dG_i = scale c_i q_i.(S dY_i) - beta_i c_i k_i.(S R_i) - gamma_i k_i.(D U_i) + sum_j N_ij - sum_j N_ji,
//   of the chunk's last frame also sum_j gamma_j k_j.(D U_j) + c_C <D, S>;  dg is its sum over all later frames of the chunk.
//
// k_delta_backward goes through the chunks of a head from its last one, as k_delta_forward, and leaves R and D; k_delta_gradients does the rest, all chunks side by side.
// (THROUGH: as of the forward pass, but of the segments behind the first one, and with what their transitions left.)  Bound as that is: 200-214 us for the same 32 sequences.
template <typename AT, int DK, int W, bool THROUGH>
__global__ __launch_bounds__(64 * W) void k_delta_backward(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, M = C / 16, NB = C / 32, KB = DK / 32;
  typedef DeltaStage<AT, DK, 64 * W, 3> Stage;
  __shared__ typename Stage::Tiles tiles[2];
  DeltaStrip<AT, DK, W> strip(a, a.f.dv, THROUGH, THROUGH ? a.segments - 1 : a.segments);
  DeltaWhere at(a.f, strip.bh, 0, C);
  const int all_chunks = (int)((at.n + C - 1) / C), chunk0 = strip.segment * a.per, chunks = all_chunks < chunk0 + a.per ? all_chunks : chunk0 + a.per;
  const float* records = a.records + strip.number(0) * delta_record(C);
  delta_f32x4 D[2 * KB];
  if (strip.segment == a.segments - 1)
    strip.get(a.dsN ? a.dsN + strip.bh * strip.matrix() : nullptr, a.f.dk, D);
  else if (THROUGH)
    delta_zero(D);
  else
    strip.get(strip.border(strip.segment), DK, D);
  Stage stage;
  DeltaElement<AT> y[M][4];
  auto load = [&](int chunk) {
    at.to(a.f, chunk > chunk0 ? chunk : chunk0, C);
    stage.load(a, at, records + (long long)at.chunk * delta_record(C));
  };
  if (chunk0 < chunks) {
    load(chunks - 1);
    strip.load(a.dy, a.lddy, at, y);
    stage.store(tiles[chunks - 1 & 1], a.f.dk);
    load(chunks - 2);
    __syncthreads();
  }
  for (int chunk = chunks - 1; chunk >= chunk0; --chunk) {
    const typename Stage::Tiles& lds = tiles[chunk & 1];
    DeltaWhere here = at;
    here.to(a.f, chunk, C);
    delta_f32x4 E[M], R[M], KD[M];
    strip.take(y, here.count, E);
    strip.load(a.dy, a.lddy, at, y);
    stage.store(tiles[chunk + 1 & 1], a.f.dk);
    load(chunk - 2);
    if (!THROUGH) strip.put(a.dstates + strip.number(chunk) * strip.kept(), DK, D);
    delta_zero(KD);
    delta_zero(R);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      delta_bf16x8 d[3], left[NI];
      delta_parts(D[2 * b], D[2 * b + 1], d);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        lds.K.left(m * 16, b * 32, left);
        KD[m] = delta_mma(left, d, KD[m]);
      }
    }
    // dU: rows of block m / 2 from all blocks behind it
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[NI], left[3];
      delta_parts(E[2 * b], E[2 * b + 1], right);
#pragma unroll
      for (int m = 0; m < 2 * b + 2; ++m) {
        lds.TP.template transposed<3>((b + m / 2) * 32, 0, m & 1, left);
        R[m] = delta_mma(left, right, R[m]);
      }
    }
    delta_f32x4 dU[M];
#pragma unroll
    for (int m = 0; m < M; ++m) dU[m] = a.f.scale * R[m] + delta_rows(lds.powers[1], m) * KD[m];
    delta_zero(R);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[3], left[3];
      delta_parts(dU[2 * b], dU[2 * b + 1], right);
#pragma unroll
      for (int m = 0; m < 2 * b + 2; ++m) {
        lds.TP.transposed((b + m / 2) * 32, 0, m & 1, left);
        R[m] = delta_mma(left, right, R[m]);
      }
    }
    if (!THROUGH) strip.put(a.dwrites + strip.number(chunk) * C * a.f.dv, C, R);
#pragma unroll
    for (int m = 0; m < M; ++m) R[m] *= delta_rows(lds.powers[2], m);
    if (!THROUGH) strip.store(a.dv, here, R);
    const float end = lds.powers[0][C - 1];
#pragma unroll
    for (int k = 0; k < 2 * KB; ++k) D[k] *= end;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[3], left[NI];
      delta_f32x4 x[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) x[t] = a.f.scale * (delta_rows(lds.powers[0], 2 * b + t) * E[2 * b + t]);
      delta_parts(x[0], x[1], right);
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) {
        lds.Q.transposed(b * 32, (k >> 1) * 32, k & 1, left);
        D[k] = delta_mma(left, right, D[k]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) x[t] = -delta_rows(lds.powers[0], 2 * b + t) * R[2 * b + t];
      delta_parts(x[0], x[1], right);
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) {
        lds.K.transposed(b * 32, (k >> 1) * 32, k & 1, left);
        D[k] = delta_mma(left, right, D[k]);
      }
    }
    __syncthreads();
  }
  if (THROUGH)
    strip.put(strip.border(strip.segment - 1), DK, D);
  else if (strip.segment == 0)
    strip.put(a.ds0 + strip.bh * strip.matrix(), a.f.dk, D);
}

// The sum over 16 neighbouring lanes, in all of them.
__device__ __forceinline__ float delta_sum16(float v) {
  auto add = [&](auto ctrl) { v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, 0xF, 0xF, true)); };
  add(std::integral_constant<int, 0xB1>());
  add(std::integral_constant<int, 0x4E>());
  add(std::integral_constant<int, 0x141>());
  add(std::integral_constant<int, 0x140>());
  return v;
}

// One chunk of one head per workgroup, DK / 16 wavefronts with 16 columns of dQ and dK each.  The values' columns pass by 32 at a time, the next ones on their way meanwhile.
// NARROW: values of fewer than eight columns.
// Columns go into one half of LDS while products are made of the other, the operands of a product are read during the one before it, and what is chosen by an element is computed without ways of its own.  Of 48 800 clocks
// of a chunk (keys and values of 128 in bf16) 14 000 go until the first columns, Q and K are there, 19 300 into the columns, 8500 into the rows' sums, N, F and H, 3000 into the last products and 4000 into results.  The
// accumulators take a compute unit's registers, one workgroup each, which does nothing else while it waits.  T=1000, 32 ragged sequences of 8 heads: 376-398 us, 1070 MB read, 150 written (482 with one half, each operand read
// when it was wanted, and a way of its own for each element of P).  Slower: 16 wavefronts of half the columns' work, 509 for 480; the frames' and states' numbers kept in the order in which they are read, which costs the
// kernels that write them 25 us and does not help this one; a compute unit's next chunk's columns asked for during its last products, 446 for 480, but 35 for 29 where chunks are few.
template <typename AT, int DK, bool NARROW>
__global__ __launch_bounds__(DK * 4) void k_delta_gradients(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, M = C / 16, NB = C / 32, BLOCKS = delta_blocks(C), W = DK / 16, THREADS = 64 * W;
  constexpr int kTiles = BLOCKS * 4, kEach = (kTiles + W - 1) / W;                                        // of C x C, for each wavefront
  constexpr int kItems = C * 4, kTasks = (2 * kItems + THREADS - 1) / THREADS;                            // eights of 32 columns: of R and V, then of U and dY
  constexpr int kApart = THREADS * 8 / DK;
  typedef decltype(delta_load8((const AT*)nullptr, 0)) Eight8;
  struct Passing {  // of the values' columns
    DeltaTile<3, C, 32> R, U;
    DeltaTile<NI, C, 32> Y;
  };
  struct Square {
    DeltaTile<3, BLOCKS * 32, 32> F, H;
  };
  __shared__ DeltaTile<NI, C, DK> K, Q;
  __shared__ union Shared {
    Passing pass[2];
    Square square;
  } lds;
  __shared__ alignas(16) float powers[5][C];  // c, gamma, beta, G in two parts
  __shared__ alignas(16) float dots[3][W][C];
  __shared__ float rv[C], ds_of[W];
  __shared__ alignas(16) float sums[3][M][C];  // sums of 16 columns of N and of X o L, of 16 rows of N
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q4 = lane >> 4, i16 = lane & 15;
  const int chunk = blockIdx.x % a.chunks, bh = blockIdx.x / a.chunks;
  const DeltaWhere at(a.f, bh, chunk, C);
  AT *dq = (AT*)a.dq, *dk = (AT*)a.dk;
  const bool each = a.dq_each != nullptr;
  // (frames past the end)
  const long long past = a.f.T - (long long)chunk * C;
  for (int i = at.count + wave; i < C && i < past; i += W) {
    const long long row = ((long long)chunk * C + i) * a.f.B + at.b, head = row * a.f.heads + at.h;
    for (int e = lane; e < a.f.dv; e += 64) store_f32((AT*)a.dv + head * a.f.dv + e, 0.f);
    for (int e = lane; e < a.f.dk; e += 64) {
      if (each) {
        a.dq_each[head * a.f.dk + e] = a.dk_each[head * a.f.dk + e] = 0.f;
      } else {
        store_f32(dq + head * a.f.dk + e, 0.f);
        store_f32(dk + head * a.f.dk + e, 0.f);
      }
    }
    if (lane == 0) a.dg[head] = a.dbeta[head] = 0.f;
  }
  if (at.count == 0) return;
  const long long number = (long long)bh * a.chunks + chunk, matrix = (long long)DK * a.f.dv;
  const float *record = a.records + number * delta_record(C), *rL = record + delta_image(C);
  const int width = a.f.dv;
  const int my_row = wave * 16 + i16;  // of S and D
  // What passes by, from column c0 on, asked for a pass ahead.
  delta_f32x8 s, d, f[kTasks];
  Eight8 x[kTasks];
  auto load_states = [&](int c0) {
    c0 = c0 < width ? c0 : 0;  // (what is loaded on a condition is waited for)
    const unsigned state = (unsigned)(my_row * width + delta_read_col(c0 + q4 * 8, width)) * 4u;
    s = delta_load8_any<NARROW>((const float*)((const char*)(a.states + number * matrix) + state), c0 + q4 * 8, width);
    d = delta_load8_any<NARROW>((const float*)((const char*)(a.dstates + number * matrix) + state), c0 + q4 * 8, width);
  };
  auto load_frames = [&](int c0) {
    c0 = c0 < width ? c0 : 0;
#pragma unroll
    for (int n = 0; n < kTasks; ++n) {
      const int first = n * THREADS + wave * 64, which = first >= kItems, item = first + lane - which * kItems, row = item >> 2, col = c0 + (item & 3) * 8;
      if (first < 2 * kItems) {
        f[n] = delta_load8_any<NARROW>((which ? a.writes : a.dwrites) + number * C * width + (row * width + delta_read_col(col, width)), col, width);
        const AT* tensor = (const AT*)(which ? a.dy : a.f.v);
        const long long ld = which ? a.lddy : a.f.ldv;
        x[n] = delta_load8_any<NARROW>(tensor + (at.row(row < at.count ? row : at.count - 1) * ld + (long long)at.h * width + delta_read_col(col, width)), col, width);
      }
    }
  };
  load_frames(0);
  load_states(0);
  {
    const int col = threadIdx.x % (DK / 8) * 8;
    for (int row = threadIdx.x / (DK / 8); row < C; row += kApart) {
      const long long r = at.row(row < at.count ? row : at.count - 1);
      delta_bf16x8 parts[NI];
      delta_parts(delta_placed<(DK <= 32)>(delta_load8_any<(DK <= 32)>((const AT*)a.f.k + (r * a.f.ldk + at.kh * a.f.dk + delta_read_col(col, a.f.dk)), col, a.f.dk), col, a.f.dk, row < at.count), parts);
      K.put(delta_place(row), col, parts);
      delta_parts(delta_placed<(DK <= 32)>(delta_load8_any<(DK <= 32)>((const AT*)a.f.q + (r * a.f.ldq + at.kh * a.f.dk + delta_read_col(col, a.f.dk)), col, a.f.dk), col, a.f.dk, row < at.count), parts);
      Q.put(delta_place(row), col, parts);
    }
  }
  for (int i = threadIdx.x; i < 5 * C; i += THREADS) powers[i / C][i % C] = rL[BLOCKS * 1024 + i];

  delta_f32x4 YS[M], UD[M], RS[M], X[kEach], Z[kEach];
  delta_zero(YS);
  delta_zero(UD);
  delta_zero(RS);
  delta_zero(X);
  delta_zero(Z);
  float ds = 0.f, own_rv[kTasks] = {};
  auto tile_m = [](int tile) { return (tile >> 2 > 0) * 2 + (tile >> 1 & 1); };
  auto tile_o = [](int tile) { return (tile >> 2 > 1) * 2 + (tile & 1); };
  auto put_frames = [&](int c0, Passing& to) {
    const bool whole = c0 + 32 <= width && at.count == C;
#pragma unroll
    for (int n = 0; n < kTasks; ++n) {
      const int first = n * THREADS + wave * 64, which = first >= kItems, item = first + lane - which * kItems, row = item >> 2, c8 = (item & 3) * 8;
      if (first < 2 * kItems) {
        if (!whole) {
          f[n] = delta_placed<NARROW>(f[n], c0 + c8, width, true);
          x[n] = delta_placed<NARROW>(x[n], c0 + c8, width, row < at.count);
        }
        delta_bf16x8 parts[3], some[NI];
        delta_parts(f[n], parts);
        (which ? to.U : to.R).put(delta_place(row), c8, parts);
        if (which) {
          delta_parts(x[n], some);
          to.Y.put(delta_place(row), c8, some);
        } else {
          const delta_f32x8 v = delta_wide(x[n]);
#pragma unroll
          for (int j = 0; j < 8; ++j) own_rv[n] = __builtin_fmaf(f[n][j], v[j], own_rv[n]);
        }
      }
    }
    load_frames(c0 + 32);
  };
  delta_bf16x8 sp[3], dp[3];
  auto take_states = [&](int c0) {
    if (c0 + 32 > width) {
      s = delta_placed<NARROW>(s, c0 + q4 * 8, width, true);
      d = delta_placed<NARROW>(d, c0 + q4 * 8, width, true);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ds = __builtin_fmaf(s[j], d[j], ds);
    delta_parts(s, sp);
    delta_parts(d, dp);
    load_states(c0 + 32);
  };
  auto products = [&](const Passing& of) {
    // (the operands of a step are read during the one before it)
    delta_bf16x8 of_Y[2][NI], of_U[2][3], of_R[2][3];
    auto fetch = [&](int step) {
      const int tile = (step - M) * W + wave, at = step & 1, some = kTiles % W == 0 || tile < kTiles ? tile : 0;
      const int m = step < M ? step : tile_m(some), o = step < M ? step : tile_o(some);
      of.Y.left(m * 16, 0, of_Y[at]);
      of.U.left(o * 16, 0, of_U[at]);
      of.R.left(m * 16, 0, of_R[at]);
    };
    fetch(0);
#pragma unroll
    for (int step = 0; step < M + kEach; ++step) {
      const int at = step & 1;
      if (step + 1 < M + kEach) fetch(step + 1);
      delta_ahead();
      if (step < M) {
        YS[step % M] = delta_mma(of_Y[at], sp, YS[step % M]);
        UD[step % M] = delta_mma(of_U[at], dp, UD[step % M]);
        RS[step % M] = delta_mma(of_R[at], sp, RS[step % M]);
      } else if (kTiles % W == 0 || (step - M) * W + wave < kTiles) {
        const int n = (step + kEach - M) % kEach;
        X[n] = delta_mma(of_R[at], of_U[at], X[n]);
        Z[n] = delta_mma(of_Y[at], of_U[at], Z[n]);
      }
    }
  };
  put_frames(0, lds.pass[0]);
  take_states(0);
  __syncthreads();
  int now = 0;
  for (int c0 = 32; c0 < width; c0 += 32, now ^= 1) {
    put_frames(c0, lds.pass[now ^ 1]);
    products(lds.pass[now]);
    take_states(c0);
    __syncthreads();
  }
  products(lds.pass[now]);
  __syncthreads();
  // P and L, all of a lane's at once, before the rows' sums
  unsigned short of_P[kEach][4][3];
  float of_L[kEach][4];
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int tile = kTiles % W == 0 || n * W + wave < kTiles ? n * W + wave : 0, block = tile >> 2, m = tile_m(tile), o = tile_o(tile);
    const int j = (i16 >> 2) * 8 + (o & 1) * 4 + (i16 & 3);  // (row and column of the block)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const char* image = (const char*)record + 3 * BLOCKS * 2048 + DeltaTile<3, BLOCKS * 32, 32>::offset(block * 32 + (m & 1) * 16 + q4 * 4 + r, j);
#pragma unroll
      for (int k = 0; k < 3; ++k) of_P[n][r][k] = *(const unsigned short*)(image + k * BLOCKS * 2048);
      of_L[n][r] = rL[block * 1024 + (q4 * 8 + (m & 1) * 4 + r) * 32 + j];
    }
  }
#pragma unroll
  for (int n = 0; n < kTasks; ++n) {
    const int first = n * THREADS + wave * 64, item = first + lane;
    if (first < kItems) {
      float v = own_rv[n];
      v += __shfl_xor(v, 1);
      v += __shfl_xor(v, 2);
      if ((item & 3) == 0) rv[item >> 2] = v;
    }
  }
  // dots of rows, and factors
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const delta_f32x4 qv = Q.of_result(m * 16, wave * 16), kv = K.of_result(m * 16, wave * 16);
    const int first = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4;
    delta_f32x4 x = qv * YS[m], y = kv * RS[m], z = kv * UD[m];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = delta_sum16(x[r]), y[r] = delta_sum16(y[r]), z[r] = delta_sum16(z[r]);
    if (i16 == 0) *(delta_f32x4*)&dots[0][wave][first] = x, *(delta_f32x4*)&dots[1][wave][first] = y, *(delta_f32x4*)&dots[2][wave][first] = z;
    const delta_f32x4 c = delta_rows(powers[0], m), gamma = delta_rows(powers[1], m), beta = delta_rows(powers[2], m);
    YS[m] *= a.f.scale * c;
    UD[m] = gamma * UD[m] - beta * c * RS[m];
  }
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int tile = n * W + wave, block = tile >> 2;
    if (kTiles % W == 0 || tile < kTiles) {
      const int m = tile_m(tile), o = tile_o(tile);
      const int j = (o >> 1) * 32 + (i16 >> 2) * 8 + (o & 1) * 4 + (i16 & 3);
      float column = 0.f;
      delta_f32x4 row, with_l;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4 + r, place = block * 32 + (m & 1) * 16 + q4 * 4 + r;
        float p = 0.f;
#pragma unroll
        for (int k = 2; k >= 0; --k) p += __builtin_bit_cast(float, (unsigned)of_P[n][r][k] << 16);
        const float l = of_L[n][r], beta = powers[2][i];
        const float power = expf(i >= j ? (powers[3][i] - powers[3][j]) + (powers[4][i] - powers[4][j]) : 0.f);  // (not on a condition, which would be a way of its own for each)
        const float x = i > j ? X[n][r] : 0.f, z = i >= j ? a.f.scale * Z[n][r] : 0.f, e = i >= j ? power : 0.f;
        const float both = z * p - x * (beta * l);
        column += both;
        row[r] = delta_sum16(both), with_l[r] = delta_sum16(x * l);
        float f = z * e, h = -(x * beta * e);
        const int to = DeltaTile<3, BLOCKS * 32, 32>::offset(place, j & 31);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const __bf16 fp = (__bf16)f, hp = (__bf16)h;
          *(__bf16*)(lds.square.F.bytes[k] + to) = fp;
          *(__bf16*)(lds.square.H.bytes[k] + to) = hp;
          f -= (float)fp, h -= (float)hp;
        }
      }
      const int first = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4;
      if (i16 == 0) *(delta_f32x4*)&sums[0][o][first] = row, *(delta_f32x4*)&sums[1][o][first] = with_l;
      column += __shfl_xor(column, 16);
      column += __shfl_xor(column, 32);
      if (q4 == 0) sums[2][m][j] = column;
    }
  }
  ds = delta_sum16(ds);
  ds += __shfl_xor(ds, 16);
  ds += __shfl_xor(ds, 32);
  if (lane == 0) ds_of[wave] = ds;
  __syncthreads();
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    delta_bf16x8 k_right[NI], q_right[NI], left[3];
    K.right(b * 32, wave * 16, k_right);
    Q.right(b * 32, wave * 16, q_right);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if (m / 2 >= b) {
        const int place = (m / 2 + b) * 32 + (m & 1) * 16;
        lds.square.F.left(place, 0, left);
        YS[m] = delta_mma(left, k_right, YS[m]);
        lds.square.H.left(place, 0, left);
        UD[m] = delta_mma(left, k_right, UD[m]);
      }
      if (m / 2 <= b) {
        lds.square.F.transposed((b + m / 2) * 32, 0, m & 1, left);
        UD[m] = delta_mma(left, q_right, UD[m]);
        lds.square.H.transposed((b + m / 2) * 32, 0, m & 1, left);
        UD[m] = delta_mma(left, k_right, UD[m]);
      }
    }
  }
  const int col = wave * 16 + i16;
  if (each) {
    if (col < a.f.dk)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4 + r;
          const long long to = (at.row(i) * a.f.heads + at.h) * a.f.dk + col;
          if (at.count == C || i < at.count) a.dq_each[to] = YS[m][r], a.dk_each[to] = UD[m][r];
        }
  } else {
    const DeltaFrames<AT, 24> to_q(a.f, dq, at, (long long)a.f.heads * a.f.dk, (long long)at.h * a.f.dk), to_k(a.f, dk, at, (long long)a.f.heads * a.f.dk, (long long)at.h * a.f.dk);
    const unsigned to = to_q.lane(q4 * 8, col);
    if (col < a.f.dk)
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = (m >> 1) * 32 + (m & 1) * 4 + r;
          if (at.count == C || i + q4 * 8 < at.count) {
            store_f32((AT*)(to_q.at(i) + to), YS[m][r]);
            store_f32((AT*)(to_k.at(i) + to), UD[m][r]);
          }
        }
  }
  if (wave == 0) {
    const int i = lane < C ? lane : 0, block = i >> 5;
    float x = 0.f, y = 0.f, z = 0.f, all = 0.f, row = 0.f, with_l = 0.f, column = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) x += dots[0][w][i], y += dots[1][w][i], z += dots[2][w][i], all += ds_of[w];
#pragma unroll
    for (int o = 0; o < M; ++o) {
      row += o < 2 * block + 2 ? sums[0][o][i] : 0.f, with_l += o < 2 * block + 2 ? sums[1][o][i] : 0.f;
      column += o >= 2 * block ? sums[2][o][i] : 0.f;
    }
    const float c = powers[0][i], gamma = powers[1][i], beta = powers[2][i];
    float end = lane < C ? gamma * z : 0.f;
    float d = lane < C ? a.f.scale * c * x - beta * c * y - gamma * z + (row - column) : 0.f;
    end = delta_sum16(end);
    end += __shfl_xor(end, 16);
    end += __shfl_xor(end, 32);
    end += powers[0][C - 1] * all;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const float o = __shfl_down(d, step);
      if (lane + step < 64) d += o;
    }
    if (lane < at.count) {
      const long long to = at.row(lane) * a.f.heads + at.h;
      a.dg[to] = d + end;
      a.dbeta[to] = rv[lane] - c * y - with_l;
    }
  }
}

// Gradients of shared queries and keys: sums over the heads that share them, in the order of these.
template <typename AT>
__global__ __launch_bounds__(256) void k_delta_shared(DeltaChunkArgs a) {
  const long long rows = a.f.T * a.f.B * a.f.key_heads, item = blockIdx.x * 256ll + threadIdx.x;
  const long long r = item / a.f.dk, e = item - r * a.f.dk;
  if (r >= rows) return;
  const int share = a.f.heads / a.f.key_heads;
  const float *q = a.dq_each + (r * share) * a.f.dk + e, *k = a.dk_each + (r * share) * a.f.dk + e;
  float dq = 0.f, dk = 0.f;
  for (int s = 0; s < share; ++s) dq += q[(long long)s * a.f.dk], dk += k[(long long)s * a.f.dk];
  store_f32((AT*)a.dq + r * a.f.dk + e, dq);
  store_f32((AT*)a.dk + r * a.f.dk + e, dk);
}

}  // namespace rtn
