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
// pass over it: S_t^T q = a S_{t-1}^T q + (k.q) u.
template <typename AT, int R>
__global__ __launch_bounds__(256) void k_delta_steps(DeltaArgs a) {
  __shared__ float parts[2][4][16][9];
  const int strips = (a.dv + 63) / 64, strip = blockIdx.x % strips, bh = blockIdx.x / strips, b = bh / a.heads, h = bh - b * a.heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = strip * 64 + (lane & 15) * 4, row = (wave * 4 + (lane >> 4)) * R;
  const int kh = h / (a.heads / a.key_heads);
  const long long n = frames_of(a.lens, b, a.T);
  const long long matrix = ((long long)b * a.heads + h) * a.dk * a.dv;
  const bool whole = col + 4 <= a.dv;
  float S[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const long long at = matrix + (long long)(row + i) * a.dv + col;
    const bool in = a.s0 && row + i < a.dk;
    if (in && whole) {
      const delta_f32x4 w = *(const delta_f32x4_any*)(a.s0 + at);
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = w[c];
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = in && col + c < a.dv ? a.s0[at + c] : 0.f;
    }
  }
  for (long long p = 0; p < n; ++p) {
    const long long t = a.reverse ? n - 1 - p : p, frame = t * a.B + b;
    float k[R], q[R], v[4];
    const AT *kp = (const AT*)a.k + frame * a.ldk + kh * a.dk, *qp = (const AT*)a.q + frame * a.ldq + kh * a.dk, *vp = (const AT*)a.v + frame * a.ldv + h * a.dv;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool in = row + i < a.dk;
      k[i] = in ? load_f32(kp + row + i) : 0.f;
      q[i] = in ? load_f32(qp + row + i) : 0.f;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = col + c < a.dv ? load_f32(vp + col + c) : 0.f;
    const float decay = expf(a.g[frame * a.heads + h]), beta = a.beta[frame * a.heads + h];
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
// those products of parts that count: with all whose order is below 3, 2^-24 of it is lost.
//
// Where a matrix of 32 rows comes out of 16 x 16 tiles and goes into the next product as its right operand, nothing is moved: lane (quarter q, i) has column i
// and, of tile t, rows 4 q + r; the operand wants rows 8 q + 0..7 of it.  So tile t is made of rows 8 q + 4 t + r, which its left operand's lane i = 4 q + r reads.  Left operands lie in LDS
// with rows in that order (position 16 t + 4 q + r), so that a tile's are neighbours.
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 delta_bf16x8;
typedef delta_bf16x8 __attribute__((aligned(2))) delta_bf16x8_any;
typedef __attribute__((__vector_size__(8 * sizeof(float)))) float delta_f32x8;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short delta_s16x4;

template <typename AT>
struct DeltaChunk;
template <>
struct DeltaChunk<__bf16> {
  static constexpr int kFrames = 64, kInput = 1, kOut = 2;  // frames; parts of an input, and order up to which products count that end in a result of the input's type
};
template <>
struct DeltaChunk<float> {
  static constexpr int kFrames = 32, kInput = 3, kOut = 3;  // (K and Q in three parts: 32 frames are what fits into LDS)
};
constexpr int delta_blocks(int frames) { return frames == 64 ? 3 : 1; }  // of 32 x 32, of a lower triangular matrix
// What is kept of a chunk: T, P, L in blocks (0,0), (1,0), (1,1), row-major; then c, gamma, beta, and G in two parts.
constexpr int delta_record(int frames) { return 3 * delta_blocks(frames) * 1024 + 5 * frames; }

struct DeltaChunkArgs {
  DeltaArgs f;
  int chunks;      // of T frames
  float* records;  // [B,heads,chunks][record]
  float* states;   // [B,heads,chunks][dk][dv] before each chunk, or NULL
  float* writes;   // [B,heads,chunks][C][dv]: U, or NULL
  const void* dy;
  long long lddy;
  const float* dsN;
  float *dstates, *dwrites;  // as states (behind each chunk) and writes (of diag(beta)'s right side), of the gradient
  void *dq, *dk, *dv;
  float *dq_each, *dk_each;  // [T,B,heads,dk], where heads share queries and keys
  float *dg, *dbeta, *ds0;
};

__device__ __forceinline__ int delta_place(int row) { return (row & ~31) | ((row >> 2 & 1) << 4) | ((row >> 3 & 3) << 2) | (row & 3); }

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
template <int ORDER, int NA, int NB>
__device__ __forceinline__ delta_f32x4 delta_mma(const delta_bf16x8 (&a)[NA], const delta_bf16x8 (&b)[NB], delta_f32x4 c) {
#pragma unroll
  for (int s = ORDER - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i <= s; ++i)
      if (i < NA && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
  return c;
}

// A matrix in LDS as N planes of R rows.
template <int N, int R, int PITCH>
struct DeltaTile {
  alignas(16) char bytes[N][R * PITCH];
  __device__ __forceinline__ void put(int place, int col, const delta_bf16x8 (&p)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) *(delta_bf16x8_any*)(bytes[n] + place * PITCH + col * 2) = p[n];
  }
  // Left operand, 16 rows from `place` on and 32 columns from `col` on.  (Or a right operand, of the transposed matrix.)
  template <int M>
  __device__ __forceinline__ void left(int place, int col, delta_bf16x8 (&p)[M]) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < M; ++n) p[n] = *(const delta_bf16x8*)(bytes[n] + (place + (lane & 15)) * PITCH + (col + (lane >> 4) * 8) * 2);
  }
  // Left operand of the transposed matrix: rows are the columns 8 q + 4 t + r of the 32 from `col` on, columns the 32 rows from `place` on.
  template <int M>
  __device__ __forceinline__ void transposed(int place, int col, int t, delta_bf16x8 (&p)[M]) const {
    across(place, col + 4 * t, 8, p);
  }
  // Right operand: the 32 rows from `place` on, the 16 columns from `col` on.
  template <int M>
  __device__ __forceinline__ void right(int place, int col, delta_bf16x8 (&p)[M]) const {
    across(place, col, 4, p);
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
    const char* at = bytes[n] + (place + (lane >> 4) * 4 + (i >> 2)) * PITCH + (col + step * (i & 3)) * 2;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) delta_s16x4*)at);
  }
  template <int M>
  __device__ __forceinline__ void across(int place, int col, int step, delta_bf16x8 (&p)[M]) const {
#pragma unroll
    for (int n = 0; n < M; ++n) {
      const delta_s16x4 a = four(n, place, col, step), b = four(n, place + 16, col, step);
      p[n] = __builtin_bit_cast(delta_bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};
// Pitches that spread 16 rows over all banks: an odd number of 16 bytes; 3 more than a multiple of 128 elements: the transposed reads' four rows and four places too.
constexpr int delta_pitch(int width) { return width * 2 + (width == 32 ? 16 : 48); }

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
// The frames of a chunk in a tensor: where the first one's `width` elements of a head are, and how far apart frames are, in elements.
template <typename T>
struct DeltaFrames {
  T* base;
  long long pitch;
  __device__ __forceinline__ DeltaFrames(T* tensor, const DeltaWhere& at, long long ld, long long head) : base(tensor + at.first * ld + head), pitch(at.step * ld) {
    asm("" : "+s"(pitch));  // (its multiples are computed where they are used: kept from chunk to chunk they do not fit into the scalar registers)
  }
};
// Elements i * pitch of a result's lane: rows 8 q + i of 32, and its column.
__device__ __forceinline__ long long delta_lane(long long pitch, int col) { return (threadIdx.x >> 4 & 3) * 8 * pitch + col; }

// T, P, L and the powers of a chunk, one workgroup of C / 16 wavefronts each, which have 16 rows of L and P each.  The inverse: diagonal blocks of 16 row by row, a column per
// lane; then T_21 = - T_22 A_21 T_11 for blocks of 16 and of 32, in float32 matrix instructions.
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
  float *rT = record, *rP = rT + BLOCKS * 1024, *rL = rP + BLOCKS * 1024, *rc = rL + BLOCKS * 1024;
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
  auto fetch = [&](const void* base, long long ld, int row, delta_bf16x8(&p)[DK / 32][NI]) {
    const DeltaFrames<const AT> frames((const AT*)base, at, ld, at.kh * a.f.dk);
    const AT* r = frames.base + (row < at.count ? row : 0) * frames.pitch + q4 * 8;
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
        kk = delta_mma<3>(kf[b], other[b], kk);
        qk = delta_mma<3>(qf[b], other[b], qk);
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
      if (nt / 2 <= wave / 2) {
        rP[block * 1024 + (i & 31) * 32 + (j & 31)] = p;
        rL[block * 1024 + (i & 31) * 32 + (j & 31)] = l;
      }
    }
  }
  __syncthreads();
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
  for (int e = threadIdx.x; e < BLOCKS * 1024; e += C * 4) {
    const int block = e >> 10, i = (e >> 5 & 31) + (block > 0) * 32, j = (e & 31) + (block > 1) * 32;
    rT[e] = X[i * ROW + j];
  }
}

// What the kernels that go through a head's chunks load of one into LDS, by way of registers, so that the next chunk's are on their way while one is worked on.
template <typename AT, int DK, int THREADS, int NP>
struct DeltaStage {
  static constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, BLOCKS = delta_blocks(C);
  static constexpr int kRows = (C * DK / 8 + THREADS - 1) / THREADS, kBlocks = (BLOCKS * 128 + THREADS - 1) / THREADS;
  typedef decltype(delta_load8((const AT*)nullptr, 0)) Eight8;
  struct Tiles {
    DeltaTile<NI, C, delta_pitch(DK)> K, Q;
    DeltaTile<3, BLOCKS * 32, delta_pitch(32)> T;
    DeltaTile<NP, BLOCKS * 32, delta_pitch(32)> P;
    alignas(16) float powers[3][C];  // c, gamma, beta
  };
  static constexpr int kApart = THREADS * 8 / DK, kPowers = (3 * C + THREADS - 1) / THREADS;  // rows from one of a thread's to the next
  static_assert(THREADS % (DK / 8) == 0, "a thread's rows have the same columns");
  Eight8 k[kRows], q[kRows];
  delta_f32x8 t[kBlocks], p[kBlocks];
  float power[kPowers];
  int count;
  // Nothing here depends on a condition of a lane, so that nothing waits: rows past the end are read as the last one and put as 0; the last eight columns of a row are read, and put,
  // where the row has them, some of them twice.  (Heads of up to 32 may have fewer than eight: column by column.)
  static __device__ __forceinline__ Eight8 eight(const AT* row, int dk) {
    if constexpr (DK > 32) {
      return delta_load8(row, 8);
    } else {
      const int col = column(dk);
      Eight8 x;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = row[col + j < dk ? j : dk - 1 - col];
      return x;
    }
  }
  static __device__ __forceinline__ int column(int dk) {
    const int col = threadIdx.x % (DK / 8) * 8;
    return DK > 32 && col > dk - 8 ? dk - 8 : col;
  }
  __device__ __forceinline__ void load(const DeltaChunkArgs& a, const DeltaWhere& at, const float* record) {
    count = at.count;
    const DeltaFrames<const AT> kf((const AT*)a.f.k, at, a.f.ldk, at.kh * a.f.dk), qf((const AT*)a.f.q, at, a.f.ldq, at.kh * a.f.dk);
    const int row = row_of(0), col = column(a.f.dk);
    if (count == C) {
      const long long k_lane = row * kf.pitch + col, q_lane = row * qf.pitch + col;
#pragma unroll
      for (int n = 0; n < kRows; ++n) {
        k[n] = eight(kf.base + n * kApart % C * kf.pitch + k_lane, a.f.dk);
        q[n] = eight(qf.base + n * kApart % C * qf.pitch + q_lane, a.f.dk);
      }
    } else {
#pragma unroll
      for (int n = 0; n < kRows; ++n) {
        const int of = row_of(n) < count ? row_of(n) : count - 1;
        k[n] = eight(kf.base + (of * kf.pitch + col), a.f.dk);
        q[n] = eight(qf.base + (of * qf.pitch + col), a.f.dk);
      }
    }
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      t[n] = delta_load8(record + item_of(n) * 8, 8);
      p[n] = delta_load8(record + BLOCKS * 1024 + item_of(n) * 8, 8);
    }
#pragma unroll
    for (int n = 0; n < kPowers; ++n) power[n] = record[3 * BLOCKS * 1024 + power_of(n)];
  }
  static __device__ __forceinline__ int row_of(int n) { return (threadIdx.x / (DK / 8) + n * kApart) % C; }  // (where threads are more than there is, some do the same)
  static __device__ __forceinline__ int item_of(int n) {
    const int item = n * THREADS + threadIdx.x;
    return BLOCKS * 128 % THREADS == 0 || item < BLOCKS * 128 ? item : BLOCKS * 128 - 1;
  }
  static __device__ __forceinline__ int power_of(int n) {
    const int item = n * THREADS + threadIdx.x;
    return 3 * C % THREADS == 0 || item < 3 * C ? item : 3 * C - 1;
  }
  __device__ __forceinline__ void store(Tiles& to, int dk) const {
    const int col = column(dk);
    auto rows = [&](auto whole) {
#pragma unroll
      for (int n = 0; n < kRows; ++n) {
        Eight8 x = k[n], y = q[n];
        if constexpr (DK == 32 || !decltype(whole)::value) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool in = row_of(n) < count && (DK > 32 || col + j < dk);
            x[j] = in ? x[j] : 0, y[j] = in ? y[j] : 0;
          }
        }
        delta_bf16x8 parts[NI];
        delta_parts(x, parts);
        to.K.put(delta_place(row_of(n)), col, parts);
        delta_parts(y, parts);
        to.Q.put(delta_place(row_of(n)), col, parts);
      }
    };
    if (count == C)
      rows(std::true_type());
    else
      rows(std::false_type());
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      const int row = item_of(n) >> 2, c8 = (item_of(n) & 3) * 8;
      delta_bf16x8 three[3], some[NP];
      delta_parts(t[n], three);
      to.T.put(delta_place(row), c8, three);
      delta_parts(p[n], some);
      to.P.put(delta_place(row), c8, some);
    }
#pragma unroll
    for (int n = 0; n < kPowers; ++n) (&to.powers[0][0])[power_of(n)] = power[n];
  }
  // Columns that no row has: 0 from the start.
  static __device__ __forceinline__ void clear(Tiles& to, int dk) {
    if (DK > 32 && dk < DK) {
      for (int item = threadIdx.x; item < NI * C * DK; item += THREADS) {
        const int n = item / (C * DK), row = item / DK % C, col = item % DK;
        if (col >= dk) *(__bf16*)(to.K.bytes[n] + row * delta_pitch(DK) + col * 2) = *(__bf16*)(to.Q.bytes[n] + row * delta_pitch(DK) + col * 2) = (__bf16)0.f;
      }
    }
  }
};
// Four rows' numbers of tile m.
__device__ __forceinline__ delta_f32x4 delta_rows(const float* of, int m) { return *(const delta_f32x4*)(of + (m >> 1) * 32 + ((threadIdx.x >> 4) & 3) * 8 + (m & 1) * 4); }

// Sixteen columns of a head's state per wavefront, in its registers, W wavefronts per workgroup, which share K, Q, T and P in LDS.
template <typename AT, int DK, int W, bool KEEP>
__global__ __launch_bounds__(64 * W) void k_delta_forward(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, OUT = DeltaChunk<AT>::kOut, M = C / 16, NB = C / 32, KB = DK / 32;
  typedef DeltaStage<AT, DK, 64 * W, OUT> Stage;
  __shared__ typename Stage::Tiles lds;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4, i16 = lane & 15;
  const int strips = (a.f.dv + 16 * W - 1) / (16 * W), strip = blockIdx.x % strips, bh = blockIdx.x / strips;
  const int col = (strip * W + wave) * 16 + i16;
  const bool has = col < a.f.dv;
  DeltaWhere at(a.f, bh, 0, C);
  const int chunks = (int)((at.n + C - 1) / C);
  const float* record = a.records + (long long)bh * a.chunks * delta_record(C);
  const long long matrix = (long long)a.f.dk * a.f.dv;
  delta_f32x4 S[2 * KB];
  auto first_of = [](int tile) { return (tile >> 1) * 32 + (tile & 1) * 4; };
  auto row_of = [&](int tile, int r) { return first_of(tile) + q4 * 8 + r; };
#pragma unroll
  for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
    for (int r = 0; r < 4; ++r) S[k][r] = a.f.s0 && has && row_of(k, r) < a.f.dk ? a.f.s0[bh * matrix + (long long)row_of(k, r) * a.f.dv + col] : 0.f;
  const long long lane_state = delta_lane(a.f.dv, col);
  const bool all_rows = a.f.dk == DK;
  long long pitch_state = a.f.dv;
  auto put_state = [&](float* to) {
    if (!has) return;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      float* row = to + b * 32 * pitch_state;
#pragma unroll
      for (int j = 0; j < 8; ++j, row += pitch_state)
        if (all_rows || b * 32 + q4 * 8 + j < a.f.dk) row[lane_state] = S[2 * b + (j >> 2)][j & 3];
    }
  };
  Stage stage;
  Stage::clear(lds, a.f.dk);
  AT v[M][4];
  auto load = [&]() {
    stage.load(a, at, record);
    const DeltaFrames<const AT> frames((const AT*)a.f.v, at, a.f.ldv, (long long)at.h * a.f.dv);
    const int of = has ? col : a.f.dv - 1;  // (what is no column is computed as the last one, and what is no row is read as the last one and taken as 0)
    if (at.count == C) {
      const long long lane_in = delta_lane(frames.pitch, of);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const AT* from = frames.base + b * 32 * frames.pitch;
#pragma unroll
        for (int j = 0; j < 8; ++j, from += frames.pitch) v[2 * b + (j >> 2)][j & 3] = from[lane_in];
      }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[m][r] = frames.base[(row_of(m, r) < at.count ? row_of(m, r) : at.count - 1) * frames.pitch + of];
    }
  };
  if (chunks) load();
  for (int chunk = 0; chunk < chunks; ++chunk) {
    const DeltaWhere here = at;
    asm("" : "+s"(pitch_state));
    delta_f32x4 R[M], O[M];
    __syncthreads();
    stage.store(lds, a.f.dk);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        R[m][r] = load_f32(&v[m][r]);
        if (here.count < C) R[m][r] = row_of(m, r) < here.count ? R[m][r] : 0.f;
      }
    __syncthreads();
    if (chunk + 1 < chunks) {
      at.to(a.f, chunk + 1, C);
      record += delta_record(C);
      load();
    }
    if (KEEP) put_state(a.states + ((long long)bh * a.chunks + chunk) * matrix);
    delta_f32x4 KS[M];
#pragma unroll
    for (int m = 0; m < M; ++m) KS[m] = O[m] = (delta_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      delta_bf16x8 s[3], left[NI];
      delta_parts(S[2 * b], S[2 * b + 1], s);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        lds.K.left(m * 16, b * 32, left);
        KS[m] = delta_mma<3>(left, s, KS[m]);
        lds.Q.left(m * 16, b * 32, left);
        O[m] = delta_mma<OUT>(left, s, O[m]);
      }
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const delta_f32x4 c = delta_rows(lds.powers[0], m);
      R[m] = delta_rows(lds.powers[2], m) * (R[m] - c * KS[m]);
      O[m] *= c;
    }
    delta_f32x4 U[M];
#pragma unroll
    for (int m = 0; m < M; ++m) U[m] = (delta_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[3], left[3];
      delta_parts(R[2 * b], R[2 * b + 1], right);
#pragma unroll
      for (int m = 2 * b; m < M; ++m) {
        lds.T.left((m / 2 + b) * 32 + (m & 1) * 16, 0, left);
        U[m] = delta_mma<3>(left, right, U[m]);
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[OUT], left[OUT];
      delta_parts(U[2 * b], U[2 * b + 1], right);
#pragma unroll
      for (int m = 2 * b; m < M; ++m) {
        lds.P.left((m / 2 + b) * 32 + (m & 1) * 16, 0, left);
        O[m] = delta_mma<OUT>(left, right, O[m]);
      }
    }
    if (has) {
      const DeltaFrames<AT> frames((AT*)a.f.y, here, (long long)a.f.heads * a.f.dv, (long long)here.h * a.f.dv);
      float* writes = a.writes + ((long long)bh * a.chunks + chunk) * C * a.f.dv;
      const long long lane_out = delta_lane(frames.pitch, col);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        AT* to = frames.base + b * 32 * frames.pitch;
        float* u = writes + b * 32 * pitch_state;
#pragma unroll
        for (int j = 0; j < 8; ++j, to += frames.pitch, u += pitch_state) {
          if (here.count == C || b * 32 + q4 * 8 + j < here.count) store_f32(to + lane_out, a.f.scale * O[2 * b + (j >> 2)][j & 3]);
          if (KEEP) u[lane_state] = U[2 * b + (j >> 2)][j & 3];
        }
      }
    }
    const float end = lds.powers[0][C - 1];
#pragma unroll
    for (int k = 0; k < 2 * KB; ++k) S[k] *= end;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[3], left[NI];
      delta_parts(delta_rows(lds.powers[1], 2 * b) * U[2 * b], delta_rows(lds.powers[1], 2 * b + 1) * U[2 * b + 1], right);
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) {
        lds.K.transposed(b * 32, (k >> 1) * 32, k & 1, left);
        S[k] = delta_mma<3>(left, right, S[k]);
      }
    }
  }
  put_state(a.f.sN + bh * matrix);
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
template <typename AT, int DK, int W>
__global__ __launch_bounds__(64 * W) void k_delta_backward(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, M = C / 16, NB = C / 32, KB = DK / 32;
  typedef DeltaStage<AT, DK, 64 * W, 3> Stage;
  __shared__ typename Stage::Tiles lds;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4, i16 = lane & 15;
  const int strips = (a.f.dv + 16 * W - 1) / (16 * W), strip = blockIdx.x % strips, bh = blockIdx.x / strips;
  const int col = (strip * W + wave) * 16 + i16;
  const bool has = col < a.f.dv;
  DeltaWhere at(a.f, bh, 0, C);
  const int chunks = (int)((at.n + C - 1) / C);
  const long long matrix = (long long)a.f.dk * a.f.dv;
  delta_f32x4 D[2 * KB];
  auto first_of = [](int tile) { return (tile >> 1) * 32 + (tile & 1) * 4; };
  auto row_of = [&](int tile, int r) { return first_of(tile) + q4 * 8 + r; };
#pragma unroll
  for (int k = 0; k < 2 * KB; ++k)
#pragma unroll
    for (int r = 0; r < 4; ++r) D[k][r] = a.dsN && has && row_of(k, r) < a.f.dk ? a.dsN[bh * matrix + (long long)row_of(k, r) * a.f.dv + col] : 0.f;
  const long long lane_state = delta_lane(a.f.dv, col);
  const bool all_rows = a.f.dk == DK;
  long long pitch_state = a.f.dv;
  auto put_state = [&](float* to) {
    if (!has) return;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      float* row = to + b * 32 * pitch_state;
#pragma unroll
      for (int j = 0; j < 8; ++j, row += pitch_state)
        if (all_rows || b * 32 + q4 * 8 + j < a.f.dk) row[lane_state] = D[2 * b + (j >> 2)][j & 3];
    }
  };
  Stage stage;
  Stage::clear(lds, a.f.dk);
  AT y[M][4];
  auto load = [&](int chunk) {
    at.to(a.f, chunk, C);
    stage.load(a, at, a.records + ((long long)bh * a.chunks + chunk) * delta_record(C));
    const DeltaFrames<const AT> frames((const AT*)a.dy, at, a.lddy, (long long)at.h * a.f.dv);
    const int of = has ? col : a.f.dv - 1;  // (what is no column is computed as the last one, and what is no row is read as the last one and taken as 0)
    if (at.count == C) {
      const long long lane_in = delta_lane(frames.pitch, of);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const AT* from = frames.base + b * 32 * frames.pitch;
#pragma unroll
        for (int j = 0; j < 8; ++j, from += frames.pitch) y[2 * b + (j >> 2)][j & 3] = from[lane_in];
      }
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) y[m][r] = frames.base[(row_of(m, r) < at.count ? row_of(m, r) : at.count - 1) * frames.pitch + of];
    }
  };
  if (chunks) load(chunks - 1);
  for (int chunk = chunks - 1; chunk >= 0; --chunk) {
    const DeltaWhere here = at;
    asm("" : "+s"(pitch_state));
    delta_f32x4 E[M], R[M], KD[M];
    __syncthreads();
    stage.store(lds, a.f.dk);
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        E[m][r] = load_f32(&y[m][r]);
        if (here.count < C) E[m][r] = row_of(m, r) < here.count ? E[m][r] : 0.f;
      }
    __syncthreads();
    if (chunk) load(chunk - 1);
    put_state(a.dstates + ((long long)bh * a.chunks + chunk) * matrix);
#pragma unroll
    for (int m = 0; m < M; ++m) KD[m] = R[m] = (delta_f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      delta_bf16x8 d[3], left[NI];
      delta_parts(D[2 * b], D[2 * b + 1], d);
#pragma unroll
      for (int m = 0; m < M; ++m) {
        lds.K.left(m * 16, b * 32, left);
        KD[m] = delta_mma<3>(left, d, KD[m]);
      }
    }
    // dU: rows of block m / 2 from all blocks behind it
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[NI], left[3];
      delta_parts(E[2 * b], E[2 * b + 1], right);
#pragma unroll
      for (int m = 0; m < 2 * b + 2; ++m) {
        lds.P.transposed((b + m / 2) * 32, 0, m & 1, left);
        R[m] = delta_mma<3>(left, right, R[m]);
      }
    }
    delta_f32x4 dU[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
      dU[m] = a.f.scale * R[m] + delta_rows(lds.powers[1], m) * KD[m];
      R[m] = (delta_f32x4){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      delta_bf16x8 right[3], left[3];
      delta_parts(dU[2 * b], dU[2 * b + 1], right);
#pragma unroll
      for (int m = 0; m < 2 * b + 2; ++m) {
        lds.T.transposed((b + m / 2) * 32, 0, m & 1, left);
        R[m] = delta_mma<3>(left, right, R[m]);
      }
    }
    if (has) {
      const DeltaFrames<AT> frames((AT*)a.dv, here, (long long)a.f.heads * a.f.dv, (long long)here.h * a.f.dv);
      float* writes = a.dwrites + ((long long)bh * a.chunks + chunk) * C * a.f.dv;
      const long long lane_out = delta_lane(frames.pitch, col);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        AT* to = frames.base + b * 32 * frames.pitch;
        float* u = writes + b * 32 * pitch_state;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const delta_f32x4 dv = delta_rows(lds.powers[2], 2 * b + t) * R[2 * b + t];
#pragma unroll
          for (int r = 0; r < 4; ++r, to += frames.pitch, u += pitch_state) {
            if (here.count == C || b * 32 + q4 * 8 + t * 4 + r < here.count) store_f32(to + lane_out, dv[r]);
            u[lane_state] = R[2 * b + t][r];
          }
        }
      }
    }
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
        D[k] = delta_mma<3>(left, right, D[k]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) x[t] = -(delta_rows(lds.powers[0], 2 * b + t) * delta_rows(lds.powers[2], 2 * b + t)) * R[2 * b + t];
      delta_parts(x[0], x[1], right);
#pragma unroll
      for (int k = 0; k < 2 * KB; ++k) {
        lds.K.transposed(b * 32, (k >> 1) * 32, k & 1, left);
        D[k] = delta_mma<3>(left, right, D[k]);
      }
    }
  }
  put_state(a.ds0 + bh * matrix);
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

// One chunk of one head per workgroup, DK / 16 wavefronts with 16 columns of dQ and dK each.  The values' columns pass by 32 at a time.
template <typename AT, int DK>
__global__ __launch_bounds__(DK * 4) void k_delta_gradients(DeltaChunkArgs a) {
  constexpr int C = DeltaChunk<AT>::kFrames, NI = DeltaChunk<AT>::kInput, OUT = DeltaChunk<AT>::kOut, M = C / 16, NB = C / 32, BLOCKS = delta_blocks(C), W = DK / 16, THREADS = 64 * W;
  constexpr int kTiles = BLOCKS * 4, kEach = (kTiles + W - 1) / W, kItems = C * 4, kOwn = (kItems + THREADS - 1) / THREADS, ROW = C + 1;
  struct Passing {  // of the values' columns
    DeltaTile<3, C, delta_pitch(32)> U, R;
    DeltaTile<NI, C, delta_pitch(32)> Y;
  };
  struct Square {
    float N[C * ROW], XL[C * ROW];
    DeltaTile<OUT, BLOCKS * 32, delta_pitch(32)> F, H;
  };
  __shared__ DeltaTile<NI, C, delta_pitch(DK)> K, Q;
  __shared__ union Shared {
    Passing pass;
    Square square;
  } lds;
  __shared__ alignas(16) float powers[5][C];  // c, gamma, beta, G in two parts
  __shared__ float dots[3][W][C], rv[C], sums[2][C], xl[C], ds_of[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q4 = lane >> 4, i16 = lane & 15;
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
  const float* record = a.records + ((long long)bh * a.chunks + chunk) * delta_record(C);
  const long long number = (long long)bh * a.chunks + chunk, matrix = (long long)a.f.dk * a.f.dv;
  const DeltaFrames<const AT> kf((const AT*)a.f.k, at, a.f.ldk, at.kh * a.f.dk), qf((const AT*)a.f.q, at, a.f.ldq, at.kh * a.f.dk);
  const DeltaFrames<const AT> vf((const AT*)a.f.v, at, a.f.ldv, (long long)at.h * a.f.dv), yf((const AT*)a.dy, at, a.lddy, (long long)at.h * a.f.dv);
  for (int item = threadIdx.x; item < C * DK / 8; item += THREADS) {
    const int row = item / (DK / 8), c8 = item % (DK / 8) * 8, left = row < at.count ? delta_left(c8, a.f.dk) : 0;
    delta_bf16x8 parts[NI];
    delta_parts(delta_load8(kf.base + (row * kf.pitch + c8), left), parts);
    K.put(delta_place(row), c8, parts);
    delta_parts(delta_load8(qf.base + (row * qf.pitch + c8), left), parts);
    Q.put(delta_place(row), c8, parts);
  }
  for (int i = threadIdx.x; i < 5 * C; i += THREADS) powers[i / C][i % C] = record[3 * BLOCKS * 1024 + i];

  const delta_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  delta_f32x4 YS[M], UD[M], RS[M], X[kEach], Z[kEach];
#pragma unroll
  for (int m = 0; m < M; ++m) YS[m] = UD[m] = RS[m] = zero;
#pragma unroll
  for (int n = 0; n < kEach; ++n) X[n] = Z[n] = zero;
  const float *U = a.writes + number * C * a.f.dv, *R = a.dwrites + number * C * a.f.dv, *S = a.states + number * matrix, *D = a.dstates + number * matrix;
  const int my_row = wave * 16 + i16;  // of S and D
  float ds = 0.f, own_rv[kOwn] = {};
  for (int c0 = 0; c0 < a.f.dv; c0 += 32) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
      const int item = n * THREADS + threadIdx.x, row = item >> 2, c8 = (item & 3) * 8;
      if (kItems % THREADS == 0 || item < kItems) {
        const int left = delta_left(c0 + c8, a.f.dv), in = row < at.count ? left : 0;
        const delta_f32x8 rr = delta_load8(R + ((long long)row * a.f.dv + c0 + c8), left);
        delta_bf16x8 parts[3], some[NI];
        delta_parts(rr, parts);
        lds.pass.R.put(delta_place(row), c8, parts);
        delta_parts(delta_load8(U + ((long long)row * a.f.dv + c0 + c8), left), parts);
        lds.pass.U.put(delta_place(row), c8, parts);
        delta_parts(delta_load8(yf.base + (row * yf.pitch + c0 + c8), in), some);
        lds.pass.Y.put(delta_place(row), c8, some);
        const delta_f32x8 v = delta_wide(delta_load8(vf.base + (row * vf.pitch + c0 + c8), in));
#pragma unroll
        for (int j = 0; j < 8; ++j) own_rv[n] = __builtin_fmaf(rr[j], v[j], own_rv[n]);
      }
    }
    const int left = my_row < a.f.dk ? delta_left(c0 + q4 * 8, a.f.dv) : 0;
    const delta_f32x8 s = delta_load8(S + ((long long)my_row * a.f.dv + c0 + q4 * 8), left), d = delta_load8(D + ((long long)my_row * a.f.dv + c0 + q4 * 8), left);
    delta_bf16x8 sp[3], dp[3];
#pragma unroll
    for (int j = 0; j < 8; ++j) ds = __builtin_fmaf(s[j], d[j], ds);
    delta_parts(s, sp);
    delta_parts(d, dp);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) {
      delta_bf16x8 left[3], some[NI];
      lds.pass.Y.left(m * 16, 0, some);
      YS[m] = delta_mma<3>(some, sp, YS[m]);
      lds.pass.U.left(m * 16, 0, left);
      UD[m] = delta_mma<3>(left, dp, UD[m]);
      lds.pass.R.left(m * 16, 0, left);
      RS[m] = delta_mma<3>(left, sp, RS[m]);
    }
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const int tile = n * W + wave, block = tile >> 2;
      if (kTiles % W == 0 || tile < kTiles) {
        const int m = (block > 0) * 2 + (tile >> 1 & 1), o = (block > 1) * 2 + (tile & 1);
        delta_bf16x8 left[3], some[NI], right[3];
        lds.pass.U.left(o * 16, 0, right);
        lds.pass.R.left(m * 16, 0, left);
        X[n] = delta_mma<3>(left, right, X[n]);
        lds.pass.Y.left(m * 16, 0, some);
        Z[n] = delta_mma<3>(some, right, Z[n]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kOwn; ++n) {
    const int item = n * THREADS + threadIdx.x;
    float v = own_rv[n];
    v += __shfl_xor(v, 1);
    v += __shfl_xor(v, 2);
    if (item < kItems && (item & 3) == 0) rv[item >> 2] = v;
  }
  for (int e = threadIdx.x; e < C * ROW; e += THREADS) lds.square.N[e] = lds.square.XL[e] = 0.f;
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int tile = n * W + wave, block = tile >> 2;
    if (kTiles % W == 0 || tile < kTiles) {
      const int m = (block > 0) * 2 + (tile >> 1 & 1), o = (block > 1) * 2 + (tile & 1);
      const int j = (o >> 1) * 32 + (i16 >> 2) * 8 + (o & 1) * 4 + (i16 & 3);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4 + r, in_block = block * 1024 + (i & 31) * 32 + (j & 31);
        const float x = i > j ? X[n][r] : 0.f, z = i >= j ? a.f.scale * Z[n][r] : 0.f;
        const float e = i >= j ? expf((powers[3][i] - powers[3][j]) + (powers[4][i] - powers[4][j])) : 0.f, beta = powers[2][i];
        const float p = record[BLOCKS * 1024 + in_block], l = record[2 * BLOCKS * 1024 + in_block];
        lds.square.N[i * ROW + j] = z * p - x * (beta * l);
        lds.square.XL[i * ROW + j] = x * l;
        const int place = block * 32 + delta_place(i & 31);
        float f = z * e, h = -(x * beta * e);
#pragma unroll
        for (int k = 0; k < OUT; ++k) {
          const __bf16 fp = (__bf16)f, hp = (__bf16)h;
          *(__bf16*)(lds.square.F.bytes[k] + place * delta_pitch(32) + (j & 31) * 2) = fp;
          *(__bf16*)(lds.square.H.bytes[k] + place * delta_pitch(32) + (j & 31) * 2) = hp;
          f -= (float)fp, h -= (float)hp;
        }
      }
    }
  }
  ds = delta_sum16(ds);
  ds += __shfl_xor(ds, 16);
  ds += __shfl_xor(ds, 32);
  if (lane == 0) ds_of[wave] = ds;
  // dots of rows, and factors
#pragma unroll
  for (int m = 0; m < M; ++m) {
    const delta_f32x4 qv = Q.of_result(m * 16, wave * 16), kv = K.of_result(m * 16, wave * 16);
    const int first = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = delta_sum16(qv[r] * YS[m][r]), y = delta_sum16(kv[r] * RS[m][r]), z = delta_sum16(kv[r] * UD[m][r]);
      if (i16 == 0) dots[0][wave][first + r] = x, dots[1][wave][first + r] = y, dots[2][wave][first + r] = z;
    }
    const delta_f32x4 c = delta_rows(powers[0], m), gamma = delta_rows(powers[1], m), beta = delta_rows(powers[2], m);
    YS[m] *= a.f.scale * c;
    UD[m] = gamma * UD[m] - beta * c * RS[m];
  }
  __syncthreads();
  // sums of rows and columns, eight threads each
  for (int item = threadIdx.x; item < C * 8; item += THREADS) {
    const int i = item >> 3, part = item & 7;
    float row = 0.f, column = 0.f, with_l = 0.f;
#pragma unroll
    for (int o = 0; o < C / 8; ++o) {
      const int j = part + 8 * o;
      row += lds.square.N[i * ROW + j], column += lds.square.N[j * ROW + i], with_l += lds.square.XL[i * ROW + j];
    }
    float d = row - column;
#pragma unroll
    for (int step = 1; step < 8; step *= 2) d += __shfl_xor(d, step), with_l += __shfl_xor(with_l, step);
    if (part == 0) sums[0][i] = d, xl[i] = with_l;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    delta_bf16x8 k_right[NI], q_right[NI], left[OUT];
    K.right(b * 32, wave * 16, k_right);
    Q.right(b * 32, wave * 16, q_right);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if (m / 2 >= b) {
        const int place = (m / 2 + b) * 32 + (m & 1) * 16;
        lds.square.F.left(place, 0, left);
        YS[m] = delta_mma<OUT>(left, k_right, YS[m]);
        lds.square.H.left(place, 0, left);
        UD[m] = delta_mma<OUT>(left, k_right, UD[m]);
      }
      if (m / 2 <= b) {
        lds.square.F.transposed((b + m / 2) * 32, 0, m & 1, left);
        UD[m] = delta_mma<OUT>(left, q_right, UD[m]);
        lds.square.H.transposed((b + m / 2) * 32, 0, m & 1, left);
        UD[m] = delta_mma<OUT>(left, k_right, UD[m]);
      }
    }
  }
  const int col = wave * 16 + i16;
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = (m >> 1) * 32 + q4 * 8 + (m & 1) * 4 + r;
      if (i < at.count && col < a.f.dk) {
        const long long to = (at.row(i) * a.f.heads + at.h) * a.f.dk + col;
        if (each) {
          a.dq_each[to] = YS[m][r], a.dk_each[to] = UD[m][r];
        } else {
          store_f32(dq + to, YS[m][r]);
          store_f32(dk + to, UD[m][r]);
        }
      }
    }
  __syncthreads();
  if (wave == 0) {
    const int i = lane < C ? lane : 0;
    float x = 0.f, y = 0.f, z = 0.f, all = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) x += dots[0][w][i], y += dots[1][w][i], z += dots[2][w][i], all += ds_of[w];
    const float c = powers[0][i], gamma = powers[1][i], beta = powers[2][i];
    float end = lane < C ? gamma * z : 0.f;
    float d = lane < C ? a.f.scale * c * x - beta * c * y - gamma * z + sums[0][i] : 0.f;
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
      a.dbeta[to] = rv[lane] - c * y - xl[lane];
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
