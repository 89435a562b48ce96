// gfx950 kernels of the gated linear recurrence and its gradient.
//
//   c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(z_t),   y_t = sigmoid(o_t) c_t
//
// Gradient, with g_t the error of c_t:  g_t = dy_t o_t + f_{t+1} g_{t+1},  dz = g i (1 - z^2),  di = g z i (1 - i),
// df = g c_{t-1} f (1 - f),  do = dy c o (1 - o)  (of the activated gates), dc0 = f_0 g_0.
#pragma once

#include "gate_functions.h"
#include "sequence_common.h"

namespace rtn {

constexpr int kRecurrenceFrames = 16;  // frames from one saved state to the next

struct RecurrenceArgs {
  const void* X;
  long long ldX;
  const float* c0;
  const int64_t* lens;
  void* Y;
  float* cN;
  float* saved;  // [chunks][B][n] the state before every kRecurrenceFrames-th frame visited
  const void* DY;
  long long ldDY;
  const float* DcN;
  void* DX;
  float* Dc0;
  long long T;
  int B, n, back;
};

// One thread per sequence and channel, frame by frame.
template <typename AT>
__global__ void k_recurrence_fwd(RecurrenceArgs a) {
  const long long id = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (id >= (long long)a.B * a.n) return;
  const int b = (int)(id / a.n), k = (int)(id % a.n);
  const long long frames = frames_of(a.lens, b, a.T);
  float c = a.c0 ? a.c0[id] : 0.f;
  for (long long s = 0; s < a.T; ++s) {
    const long long t = a.back ? a.T - 1 - s : s;
    if (a.saved && s % kRecurrenceFrames == 0) a.saved[s / kRecurrenceFrames * a.B * a.n + id] = c;
    float y = 0.f;
    if (t < frames) {
      const AT* x = (const AT*)a.X + (t * a.B + b) * a.ldX + k;
      const float z = Act<AT>::tanh(load_f32(x)), i = Act<AT>::sigmoid(load_f32(x + a.n)), f = Act<AT>::sigmoid(load_f32(x + 2 * (long long)a.n)),
                  o = Act<AT>::sigmoid(load_f32(x + 3 * (long long)a.n));
      c = __builtin_fmaf(f, c, i * z);
      y = o * c;
    }
    store_f32((AT*)a.Y + (t * a.B + b) * a.n + k, y);
  }
  a.cN[id] = c;
}

template <typename AT>
__global__ void k_recurrence_bwd(RecurrenceArgs a) {
  const long long id = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (id >= (long long)a.B * a.n) return;
  const int b = (int)(id / a.n), k = (int)(id % a.n);
  const long long frames = frames_of(a.lens, b, a.T), n = a.n;
  float g = a.DcN ? a.DcN[id] : 0.f;
  for (long long s0 = ((a.T + kRecurrenceFrames - 1) / kRecurrenceFrames - 1) * kRecurrenceFrames; s0 >= 0; s0 -= kRecurrenceFrames) {
    float before[kRecurrenceFrames], c = a.saved[s0 / kRecurrenceFrames * a.B * n + id];
#pragma unroll
    for (int j = 0; j < kRecurrenceFrames; ++j) {
      const long long s = s0 + j, t = a.back ? a.T - 1 - s : s;
      before[j] = c;
      if (s < a.T && t < frames) {
        const AT* x = (const AT*)a.X + (t * a.B + b) * a.ldX + k;
        c = __builtin_fmaf(Act<AT>::sigmoid(load_f32(x + 2 * n)), c, Act<AT>::sigmoid(load_f32(x + n)) * Act<AT>::tanh(load_f32(x)));
      }
    }
#pragma unroll
    for (int j = kRecurrenceFrames - 1; j >= 0; --j) {
      const long long s = s0 + j, t = a.back ? a.T - 1 - s : s;
      if (s >= a.T) continue;
      float dz = 0.f, di = 0.f, df = 0.f, d_o = 0.f;
      if (t < frames) {
        const AT* x = (const AT*)a.X + (t * a.B + b) * a.ldX + k;
        const float z = Act<AT>::tanh(load_f32(x)), i = Act<AT>::sigmoid(load_f32(x + n)), f = Act<AT>::sigmoid(load_f32(x + 2 * n)), o = Act<AT>::sigmoid(load_f32(x + 3 * n));
        const float dy = load_f32((const AT*)a.DY + (t * a.B + b) * a.ldDY + k);
        const float after = __builtin_fmaf(f, before[j], i * z);
        g = __builtin_fmaf(dy, o, g);
        dz = g * i * (1.f - z * z);
        di = g * z * i * (1.f - i);
        df = g * before[j] * f * (1.f - f);
        d_o = dy * after * o * (1.f - o);
        g *= f;
      }
      AT* d = (AT*)a.DX + (t * a.B + b) * 4 * n + k;
      store_f32(d, dz);
      store_f32(d + n, di);
      store_f32(d + 2 * n, df);
      store_f32(d + 3 * n, d_o);
    }
  }
  a.Dc0[id] = g;
}

}  // namespace rtn
