// gfx950 kernels of the gated delta rule: a recurrence whose state is a matrix per head.
//
//   S_t = a_t S_{t-1} + k_t u_t^T,   u_t = b_t (v_t - a_t S_{t-1}^T k_t),   o_t = s S_t^T q_t,   a_t = e^{g_t}
#pragma once

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

}  // namespace rtn
