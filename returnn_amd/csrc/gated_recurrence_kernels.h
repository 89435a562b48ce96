// gfx950 kernels of the gated linear recurrence and its gradient.
//
//   c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(z_t),   y_t = sigmoid(o_t) c_t
//
// Gradient, with g_t the error of c_t:  g_t = dy_t o_t + f_{t+1} g_{t+1},  dz = g i (1 - z^2),  di = g z i (1 - i),
// df = g c_{t-1} f (1 - f),  do = dy c o (1 - o)  (of the activated gates), dc0 = f_0 g_0.
//
// Any run of frames turns the state before it, c, into A c + S: A is the product of its forget gates, S what it would leave of a state of 0.  Runs
// after one another are joined by (A2 A1, A2 S1 + S2).  So a wavefront takes F frames of 64 lanes' channels, whose gates it holds in registers
// after reading them once; the W wavefronts of a workgroup take runs of F frames that follow each other and hand (A, S) over through LDS; and the
// workgroup goes on to the next W F frames, whose gates were asked for before the hand-over.  The gradient runs from the last frame to the first with
// (A, Q) for the errors, and the states inside a run are computed again from those that the forward pass leaves every kSavedFrames frames.
// Where sequences and channels are too few to fill the device, the frames are cut into segments: a first kernel leaves (A, S) or (A, Q) of every
// segment, and the second starts each from those before it, joined in order.  All sums are in a fixed order.
#pragma once

#include <type_traits>

#include "gate_functions.h"
#include "sequence_common.h"

namespace rtn {

constexpr int kSavedFrames = 16;  // frames from one saved state to the next
constexpr int kStreamed = 2;      // cache policy of stores: not kept in the caches

struct RecurrenceArgs {
  const void* X;
  long long ldX;
  const float* c0;  // (forward only: for the gradient it is the first of `saved`)
  const int64_t* lens;
  void* Y;
  float* cN;
  float* saved;  // [ceil(T/kSavedFrames)][B][n] the state before every kSavedFrames-th frame visited
  const void* DY;
  long long ldDY;
  const float* DcN;
  void* DX;
  float* Dc0;
  long long T;
  int B, n, back;
  int strips;         // of 64 lanes' channels, in n
  unsigned chains;    // strips times sequences
  long long segment;  // frames of a segment
  int segments;
  int apart;          // strips share no cache line
  float* runs;        // [segments][chains][64 lanes][VEC][2] A and S, or A and Q, of the segments
};

// The gates' functions, but for the hyperbolic tangent of a bfloat16 number near 0: the difference by which it is computed elsewhere is good to 2e-7,
// which may be all of the result there, while the states that it goes into are float32.  x itself leaves out x^2 / 3 of it: at |x| = 2^-7 both are good to
// 2^-15 of the result, and better on their sides of it; the cell input was rounded to 2^-9.  (With the cubic term too, below 1/16: 2e-6 of the result,
// but T=1000, 32 rows of n=1024 forward 63.7 us instead of 62.2, without either 61.8; T=16384, 2 rows of n=500 56.2, 52.5, 52.2.)
template <typename AT>
struct Gate : Act<AT> {};
template <>
struct Gate<__bf16> : Act<__bf16> {
  static __device__ __forceinline__ float tanh(float x) {
    return __builtin_fabsf(x) < 0x1p-7f ? x : Act<__bf16>::tanh(x);
  }
};

// VEC neighbouring channels of a lane: one load, at any element's address.
template <typename AT, int VEC>
struct Channels;
template <>
struct Channels<__bf16, 1> {
  typedef unsigned short Raw;
  static __device__ __forceinline__ Raw load(__amdgpu_buffer_rsrc_t row, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b16(row, at, 0, 0); }
  template <bool STREAMED>
  static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t row, unsigned at, Raw v) {
    __builtin_amdgcn_raw_buffer_store_b16(v, row, at, 0, STREAMED ? kStreamed : 0);
  }
  static __device__ __forceinline__ void get(Raw r, float (&v)[1]) { v[0] = __builtin_bit_cast(float, (unsigned)r << 16); }
  static __device__ __forceinline__ Raw set(const float (&v)[1]) { return __builtin_bit_cast(unsigned short, (__bf16)v[0]); }
};
struct OneWord {
  typedef unsigned Raw;
  static __device__ __forceinline__ Raw load(__amdgpu_buffer_rsrc_t row, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b32(row, at, 0, 0); }
  template <bool STREAMED>
  static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t row, unsigned at, Raw v) {
    __builtin_amdgcn_raw_buffer_store_b32(v, row, at, 0, STREAMED ? kStreamed : 0);
  }
};
struct TwoWords {
  typedef unsigned Raw __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ Raw load(__amdgpu_buffer_rsrc_t row, unsigned at) { return __builtin_amdgcn_raw_buffer_load_b64(row, at, 0, 0); }
  template <bool STREAMED>
  static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t row, unsigned at, Raw v) {
    __builtin_amdgcn_raw_buffer_store_b64(v, row, at, 0, STREAMED ? kStreamed : 0);
  }
};
template <>
struct Channels<float, 1> : OneWord {
  static __device__ __forceinline__ void get(Raw r, float (&v)[1]) { v[0] = __builtin_bit_cast(float, r); }
  static __device__ __forceinline__ Raw set(const float (&v)[1]) { return __builtin_bit_cast(unsigned, v[0]); }
};
template <>
struct Channels<float, 2> : TwoWords {
  static __device__ __forceinline__ void get(Raw r, float (&v)[2]) {
    v[0] = __builtin_bit_cast(float, (unsigned)r.x);
    v[1] = __builtin_bit_cast(float, (unsigned)r.y);
  }
  static __device__ __forceinline__ Raw set(const float (&v)[2]) { return Raw{__builtin_bit_cast(unsigned, v[0]), __builtin_bit_cast(unsigned, v[1])}; }
};
template <>
struct Channels<__bf16, 2> : OneWord {
  static __device__ __forceinline__ void get(Raw r, float (&v)[2]) {
    v[0] = __builtin_bit_cast(float, r << 16);
    v[1] = __builtin_bit_cast(float, r & 0xFFFF0000u);
  }
  static __device__ __forceinline__ Raw set(const float (&v)[2]) { return pack_bf16(v[0], v[1]); }
};
template <>
struct Channels<__bf16, 4> : TwoWords {
  static __device__ __forceinline__ void get(Raw r, float (&v)[4]) {
    v[0] = __builtin_bit_cast(float, (unsigned)r.x << 16);
    v[1] = __builtin_bit_cast(float, (unsigned)r.x & 0xFFFF0000u);
    v[2] = __builtin_bit_cast(float, (unsigned)r.y << 16);
    v[3] = __builtin_bit_cast(float, (unsigned)r.y & 0xFFFF0000u);
  }
  static __device__ __forceinline__ Raw set(const float (&v)[4]) { return Raw{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])}; }
};

// Rows of one sequence in an array of frames: frame t begins `frame` bytes after frame t - 1, a row has `bytes`.
struct Rows {
  char* base;
  long long frame;
  int bytes;
  __device__ __forceinline__ char* of(int t) const { return base + t * frame; }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(char* row) const { return __builtin_amdgcn_make_buffer_rsrc(row, 0, bytes, 0x00020000); }
};

// The number of the workgroup among its kernel's.  Workgroup i runs on XCD i mod 8, which has an L2 of its own.  Where neighbouring strips share cache
// lines, each XCD takes numbers that follow each other, and lines are read once and written whole (n = 1001 float32, T = 333, 11 rows: forward 27.2 / 23.8 us,
// gradient 38.9 / 33.0; n = 1000 bf16, T = 1000, 32 rows: gradient 186 / 146); where they do not, neighbours on different XCDs are a little faster (n = 1024 bf16, T = 1000, 32 rows: 69 and 118 us instead of 72 and 121).
__device__ __forceinline__ unsigned workgroup_number(const RecurrenceArgs& a) {
  const unsigned x = blockIdx.x % 8, i = blockIdx.x / 8, each = gridDim.x / 8, more = gridDim.x % 8;
  return a.apart ? blockIdx.x : x * each + (x < more ? x : more) + i;
}

// What a workgroup works on: one sequence, 64 lanes' channels, a segment of the frames.  Frames are counted in the order of the recurrence: step s is
// frame s, or T - 1 - s.
template <typename AT, int VEC>
struct Chain {
  typedef Channels<AT, VEC> C;
  typedef typename C::Raw Raw;
  int b, lane;
  unsigned k;        // the lane's first channel; lanes past the last repeat the last ones
  unsigned at[4];    // where it is in a row of gates, in bytes
  bool active;       // has channels of its own
  int low, high;     // steps inside the sequence
  int first, stride;  // frame of step 0, of the next one
  __device__ __forceinline__ Chain(const RecurrenceArgs& a, unsigned chain) {
    lane = threadIdx.x & 63;
    b = chain / a.strips;
    const unsigned own = (chain - b * a.strips) * 64 * VEC + lane * VEC;
    active = own < (unsigned)a.n;
    k = own + VEC <= (unsigned)a.n ? own : a.n - VEC;
#pragma unroll
    for (int g = 0; g < 4; ++g) at[g] = (k + g * (unsigned)a.n) * (unsigned)sizeof(AT);
    const int T = (int)a.T, frames = (int)frames_of(a.lens, b, a.T);
    low = a.back ? T - frames : 0;
    high = a.back ? T : frames;
    first = a.back ? T - 1 : 0;
    stride = a.back ? -1 : 1;
  }
  __device__ __forceinline__ bool inside(int s) const { return s >= low && s < high; }
  __device__ __forceinline__ int frame(int s) const { return first + stride * s; }
  // the frame of a step that is read in its place: itself, or one inside (there is one where any step near it is inside)
  __device__ __forceinline__ int frame_inside(int s) const {
    s = s < low ? low : s;
    return frame(s < high ? s : high - 1);
  }
  __device__ __forceinline__ bool any_inside(int s, int count) const { return s < high && s + count > low && low < high; }
  __device__ __forceinline__ bool all_inside(int s, int count) const { return s >= low && s + count <= high; }
  static __device__ __forceinline__ Rows rows(const RecurrenceArgs& a, const void* p, int b, long long ld, int width) {
    return {(char*)p + b * ld * (long long)sizeof(AT), a.B * ld * (long long)sizeof(AT), width * (int)sizeof(AT)};
  }
};

// (A, S) of a lane's channels.
template <int VEC>
struct Run {
  float a[VEC], s[VEC];
  static __device__ __forceinline__ Run none() {
    Run r;
#pragma unroll
    for (int v = 0; v < VEC; ++v) r.a[v] = 1.f, r.s[v] = 0.f;
    return r;
  }
  __device__ __forceinline__ void then(const Run& next) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = __builtin_fmaf(next.a[v], s[v], next.s[v]), a[v] *= next.a[v];
  }
  __device__ __forceinline__ void apply(float (&c)[VEC]) const {
#pragma unroll
    for (int v = 0; v < VEC; ++v) c[v] = __builtin_fmaf(a[v], c[v], s[v]);
  }
};

// The state (or error) with which segment `segment` starts, from that of the first and the segments' runs; FORWARD: those before it, else those after it.
// All wavefronts of the workgroup call this: each joins a share of the runs.
template <int VEC, int W, bool FORWARD>
__device__ __forceinline__ void start_of_segment(const RecurrenceArgs& a, unsigned chain, int segment, int wave, int lane, Run<VEC> (*shared)[64], float (&c)[VEC]) {
  const int count = FORWARD ? segment : a.segments - 1 - segment;
  if (W == 1 || count == 0) return;
  const int share = (count + W - 1) / W;
  Run<VEC> mine = Run<VEC>::none();
#pragma unroll 4
  for (int j = wave * share; j < (wave + 1) * share && j < count; ++j) {
    const int at = FORWARD ? j : a.segments - 1 - j;
    mine.then(((const Run<VEC>*)a.runs)[((size_t)at * a.chains + chain) * 64 + lane]);
  }
  shared[wave][lane] = mine;
  __syncthreads();
#pragma unroll 4
  for (int j = 0; j < W; ++j) shared[j][lane].apply(c);
  __syncthreads();
}

// Calls f with two truths as types.
template <typename F>
__device__ __forceinline__ void by_kind(bool all, bool more, F f) {
  if (all && more)
    f(std::true_type(), std::true_type());
  else if (all)
    f(std::true_type(), std::false_type());
  else if (more)
    f(std::false_type(), std::true_type());
  else
    f(std::false_type(), std::false_type());
}

// The turns of a workgroup, of `frames` steps each, that have steps of the sequence: first, first + frames, ... below stop.
struct Turns {
  int first, stop;
  template <typename C>
  __device__ __forceinline__ Turns(const C& q, int begin, int end, int frames) {
    const int low = q.low > begin ? q.low : begin, high = q.high < end ? q.high : end;
    first = low < high ? begin + (low - begin) / frames * frames : end;
    stop = low < high ? begin + (high - begin + frames - 1) / frames * frames : end;
  }
};

// ---- forward ----
// W wavefronts, F frames each.  handed: the runs of the wavefronts, and in [W] the state that the next turn starts from, which the last wavefront
// leaves there; both twice, so that one barrier a turn is enough.
// Bound by memory where there are 256 chains or more: T=1000, 32 rows of n=1024 bf16 69 us (328 MB, 4.75 TB/s; a copy of this size reaches 5.4; with gates that
// cost nothing 67), T=500, 64 rows of n=512 float32, two channels a lane, 66.5 us (4.9).  Ragged lengths save bytes but not the longest sequence's turns: 67 and 61.5 us
// with 3/4 of the gates.
template <typename AT, int VEC, int F, int W>
__global__ __launch_bounds__(64 * W) void k_recurrence_fwd(RecurrenceArgs a) {
  typedef Chain<AT, VEC> C;
  __shared__ Run<VEC> handed[2][W + 1][64];
  const unsigned number = workgroup_number(a), chain = number % a.chains;
  const int segment = number / a.chains, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const C q(a, chain);
  const int begin = segment * (int)a.segment, end = begin + (int)a.segment < (int)a.T ? begin + (int)a.segment : (int)a.T;
  const Turns turns(q, begin, end, F * W);
  const Rows X = C::rows(a, a.X, q.b, a.ldX, 4 * a.n), Y = C::rows(a, a.Y, q.b, a.n, a.n);
  const size_t own = (size_t)q.b * a.n + q.k;

  typename C::Raw raw[F][4];
  auto ask = [&](int j, char* row) {
#pragma unroll
    for (int g = 0; g < 4; ++g) raw[j][g] = C::C::load(X.at(row), q.at[g]);
  };
  if (turns.first < turns.stop && q.any_inside(turns.first + wave * F, F)) {
#pragma unroll
    for (int j = 0; j < F; ++j) ask(j, X.of(q.frame_inside(turns.first + wave * F + j)));
  }
  float c[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) c[v] = a.c0 ? a.c0[own + v] : 0.f;
  start_of_segment<VEC, W, true>(a, chain, segment, wave, q.lane, handed[0], c);

  int turn = 0;
#pragma unroll 1
  for (int from = turns.first; from < turns.stop; from += F * W, turn ^= 1) {
    const int s0 = from + wave * F, next = s0 + F * W;
    const bool all = q.all_inside(s0, F), more = next < turns.stop && q.all_inside(next, F);
    float A[F][VEC], S[F][VEC];  // of the run up to frame j
    typename C::Raw out[F];      // the output gates as they came
    by_kind(all, more, [&](auto all, auto more) {
      char* row = X.of(q.frame(next));
#pragma unroll
      for (int j = 0; j < F; ++j) {
        float z[VEC], i[VEC], f[VEC];
        C::C::get(raw[j][0], z);
        C::C::get(raw[j][1], i);
        C::C::get(raw[j][2], f);
        out[j] = raw[j][3];
        const bool in = all || q.inside(s0 + j);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float fv = in ? Gate<AT>::sigmoid(f[v]) : 1.f, iz = in ? Gate<AT>::sigmoid(i[v]) * Gate<AT>::tanh(z[v]) : 0.f;
          A[j][v] = j ? A[j - 1][v] * fv : fv;
          S[j][v] = j ? __builtin_fmaf(fv, S[j - 1][v], iz) : iz;
        }
        __builtin_amdgcn_sched_barrier(0);  // (the registers of frame j take the next turn's: the loads go on while the gates are worked on)
        if (more) ask(j, row), row += q.stride * X.frame;
      }
    });
    if (!more && next < turns.stop && q.any_inside(next, F)) {
#pragma unroll
      for (int j = 0; j < F; ++j) ask(j, X.of(q.frame_inside(next + j)));
    }
    Run<VEC> run;
#pragma unroll
    for (int v = 0; v < VEC; ++v) run.a[v] = A[F - 1][v], run.s[v] = S[F - 1][v];
    if constexpr (W > 1) {
      handed[turn][wave][q.lane] = run;
      __syncthreads();
      if (from > turns.first) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) c[v] = handed[turn][W][q.lane].s[v];
      }
#pragma unroll 4
      for (int j = 0; j < wave; ++j) handed[turn][j][q.lane].apply(c);
    }
    if (a.saved && q.active && s0 % kSavedFrames == 0 && s0 < (int)a.T) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) a.saved[(size_t)(s0 / kSavedFrames) * a.B * a.n + own + v] = c[v];
    }
    if (q.active) {
      by_kind(all, a.apart, [&](auto all, auto apart) {
        char* row = Y.of(q.frame(s0));
#pragma unroll
        for (int j = 0; j < F; ++j, row += q.stride * Y.frame) {
          if (!all && s0 + j >= end) break;
          float o[VEC], y[VEC];
          C::C::get(out[j], o);
          const bool in = all || q.inside(s0 + j);
#pragma unroll
          for (int v = 0; v < VEC; ++v) y[v] = in ? Gate<AT>::sigmoid(o[v]) * __builtin_fmaf(A[j][v], c[v], S[j][v]) : 0.f;
          C::C::template store<decltype(apart)::value>(Y.at(row), q.at[0], C::C::set(y));
        }
      });
    }
    if (W == 1 || wave == W - 1) {
      run.apply(c);
      if constexpr (W > 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) run.s[v] = c[v];
        handed[turn ^ 1][W][q.lane] = run;
      }
    }
  }
  if (!q.active) return;
  if (wave == W - 1 && segment == a.segments - 1) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) a.cN[own + v] = c[v];
  }
  // what is past the end of the sequence
  const float zero[VEC] = {};
#pragma unroll 1
  for (int s = begin + wave; s < end; s += W)
    if (s < turns.first || s >= turns.stop) C::C::template store<false>(Y.at(Y.of(q.frame(s))), q.at[0], C::C::set(zero));
}

// ---- gradient ----
// Bound by memory: T=1000, 32 rows of n=1024 bf16 118 us (590 MB, 5.0 TB/s; the simple loop over the frames 1900), T=500, 64 rows of n=512 float32 128 us (4.6).
template <typename AT, int VEC, int F, int W>
__global__ __launch_bounds__(64 * W) void k_recurrence_bwd(RecurrenceArgs a) {
  typedef Chain<AT, VEC> C;
  constexpr int GROUP = kSavedFrames / F;  // wavefronts from one saved state to the next
  static_assert(W == 1 || W % GROUP == 0, "saved states lie where wavefronts begin");
  __shared__ Run<VEC> handed[2][W + 1][64];
  __shared__ Run<VEC> states[2][W][64];
  const unsigned number = workgroup_number(a), chain = number % a.chains;
  const int segment = a.segments - 1 - (int)(number / a.chains), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const C q(a, chain);
  const int begin = segment * (int)a.segment, end = begin + (int)a.segment < (int)a.T ? begin + (int)a.segment : (int)a.T;
  const Turns turns(q, begin, end, F * W);
  const Rows X = C::rows(a, a.X, q.b, a.ldX, 4 * a.n), DY = C::rows(a, a.DY, q.b, a.ldDY, a.n), DX = C::rows(a, a.DX, q.b, 4 * (long long)a.n, 4 * a.n);
  const size_t own = (size_t)q.b * a.n + q.k;

  typename C::Raw raw[F][5];
  float before[VEC];  // the saved state of the wavefront's group
  auto ask = [&](int j, char* row, char* row_dy) {
#pragma unroll
    for (int g = 0; g < 4; ++g) raw[j][g] = C::C::load(X.at(row), q.at[g]);
    raw[j][4] = C::C::load(DY.at(row_dy), q.at[0]);
  };
  auto ask_near = [&](int s0) {
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int t = q.frame_inside(s0 + j);
      ask(j, X.of(t), DY.of(t));
    }
  };
  auto ask_state = [&](int s0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) before[v] = s0 < (int)a.T ? a.saved[(size_t)(s0 / kSavedFrames) * a.B * a.n + own + v] : 0.f;
  };
  const int last = turns.stop - F * W;
  if (turns.first < turns.stop) {
    if (q.any_inside(last + wave * F, F)) ask_near(last + wave * F);
    ask_state(last + wave * F);
  }
  float g[VEC], left[VEC];  // the error of the wavefront's last state; what the first wavefront leaves
#pragma unroll
  for (int v = 0; v < VEC; ++v) g[v] = a.DcN ? a.DcN[own + v] : 0.f;
  start_of_segment<VEC, W, false>(a, chain, segment, wave, q.lane, handed[0], g);
#pragma unroll
  for (int v = 0; v < VEC; ++v) left[v] = g[v];

  int turn = 0;
#pragma unroll 1
  for (int from = last; from >= turns.first && turns.first < turns.stop; from -= F * W, turn ^= 1) {
    const int s0 = from + wave * F, next = s0 - F * W;
    const bool all = q.all_inside(s0, F), more = from > turns.first && q.all_inside(next, F);
    float z[F][VEC], i[F][VEC], f[F][VEC], o[F][VEC], c[VEC];
    typename C::Raw error[F];  // of the outputs, as they came
    by_kind(all, more, [&](auto all, auto more) {
      char *row = X.of(q.frame(next)), *row_dy = DY.of(q.frame(next));
#pragma unroll
      for (int j = 0; j < F; ++j) {
        C::C::get(raw[j][0], z[j]);
        C::C::get(raw[j][1], i[j]);
        C::C::get(raw[j][2], f[j]);
        C::C::get(raw[j][3], o[j]);
        error[j] = raw[j][4];
        const bool in = all || q.inside(s0 + j);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          z[j][v] = in ? Gate<AT>::tanh(z[j][v]) : 0.f;
          i[j][v] = in ? Gate<AT>::sigmoid(i[j][v]) : 0.f;
          f[j][v] = in ? Gate<AT>::sigmoid(f[j][v]) : 1.f;
          o[j][v] = in ? Gate<AT>::sigmoid(o[j][v]) : 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
        if (more) ask(j, row, row_dy), row += q.stride * X.frame, row_dy += q.stride * DY.frame;
      }
    });
    if (!more && from > turns.first && q.any_inside(next, F)) ask_near(next);
    Run<VEC> forth = Run<VEC>::none(), back = forth;
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int l = F - 1 - j;
      float e[VEC];
      C::C::get(error[l], e);
      const bool in = q.inside(s0 + l);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        forth.a[v] *= f[j][v];
        forth.s[v] = __builtin_fmaf(f[j][v], forth.s[v], i[j][v] * z[j][v]);
        back.s[v] = f[l][v] * __builtin_fmaf(in ? e[v] : 0.f, o[l][v], back.s[v]);
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) back.a[v] = forth.a[v], c[v] = before[v];
    if (from > turns.first) ask_state(next);
    if constexpr (W > 1) {
      handed[turn][wave][q.lane] = back;
      states[turn][wave][q.lane] = forth;
      __syncthreads();
      if (from < last) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) g[v] = handed[turn][W][q.lane].s[v];
      }
#pragma unroll 1
      for (int j = wave / GROUP * GROUP; j < wave; ++j) states[turn][j][q.lane].apply(c);
#pragma unroll 4
      for (int j = W - 1; j > wave; --j) handed[turn][j][q.lane].apply(g);
    }
    if (wave == 0) {  // the error that the turn before this one starts from
#pragma unroll
      for (int v = 0; v < VEC; ++v) left[v] = back.s[v] = __builtin_fmaf(back.a[v], g[v], back.s[v]);
      if (W > 1) handed[turn ^ 1][W][q.lane] = back;
    }
    if (q.active) {
      float states_before[F + 1][VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        states_before[0][v] = c[v];
#pragma unroll
        for (int j = 0; j < F; ++j) states_before[j + 1][v] = __builtin_fmaf(f[j][v], states_before[j][v], i[j][v] * z[j][v]);
      }
      by_kind(all, a.apart, [&](auto all, auto apart) {
        constexpr bool STREAMED = decltype(apart)::value;  // (past the caches, but not parts of lines)
        char* row = DX.of(q.frame(s0 + F - 1));
#pragma unroll
        for (int j = F - 1; j >= 0; --j, row -= q.stride * DX.frame) {
          const bool in = all || q.inside(s0 + j);
          float e[VEC], dz[VEC], di[VEC], df[VEC], d_o[VEC];
          C::C::get(error[j], e);
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const float zv = z[j][v], iv = i[j][v], fv = f[j][v], ov = o[j][v], eo = e[v] * ov;
            const float total = g[v] + eo, gi = total * iv, gf = total * fv;
            dz[v] = in ? gi * __builtin_fmaf(-zv, zv, 1.f) : 0.f;
            di[v] = in ? gi * zv * (1.f - iv) : 0.f;
            df[v] = in ? gf * states_before[j][v] * (1.f - fv) : 0.f;
            d_o[v] = in ? eo * states_before[j + 1][v] * (1.f - ov) : 0.f;
            g[v] = in ? gf : g[v];
          }
          if (!all && s0 + j >= end) continue;
          C::C::template store<STREAMED>(DX.at(row), q.at[0], C::C::set(dz));
          C::C::template store<STREAMED>(DX.at(row), q.at[1], C::C::set(di));
          C::C::template store<STREAMED>(DX.at(row), q.at[2], C::C::set(df));
          C::C::template store<STREAMED>(DX.at(row), q.at[3], C::C::set(d_o));
        }
      });
    }
  }
  if (!q.active) return;
  if (wave == 0 && segment == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) a.Dc0[own + v] = left[v];
  }
  // what is past the end of the sequence
  const float zero[VEC] = {};
#pragma unroll 1
  for (int s = begin + wave; s < end; s += W)
    if (s < turns.first || s >= turns.stop) {
#pragma unroll
      for (int k = 0; k < 4; ++k) C::C::template store<false>(DX.at(DX.of(q.frame(s))), q.at[k], C::C::set(zero));
    }
}

// ---- the runs of segments: (A, S), or (A, Q) of the errors ----
// A wavefront takes a share of the segment's frames that follow each other, F at a time.  (Asking for the next F while these are worked on changes nothing.)
// T=16384, 2 rows of n=500 bf16, of which one has half the frames: 25 us forward, 17 in the gradient, of 62 and 80 together; T=4000, one row of n=1024: 6 of 16.
// One pass instead, in which workgroups publish their runs and look back at earlier ones, took longer (78 and 188 us): its hand-over costs more than these bytes.
template <typename AT, int VEC, int F, int W, bool FORWARD>
__global__ __launch_bounds__(64 * W) void k_recurrence_runs(RecurrenceArgs a) {
  typedef Chain<AT, VEC> C;
  __shared__ Run<VEC> handed[W][64];
  const unsigned number = workgroup_number(a), chain = number % a.chains;
  const int segment = (int)(number / a.chains) + (FORWARD ? 0 : 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (the last one's, or the first one's, nobody needs)
  const C q(a, chain);
  const int share = (int)a.segment / W, begin = segment * (int)a.segment + wave * share;
  const Rows X = C::rows(a, a.X, q.b, a.ldX, 4 * a.n), DY = C::rows(a, a.DY, q.b, a.ldDY, a.n);
  Run<VEC> run = Run<VEC>::none();
#pragma unroll 1
  for (int k = 0; k < share; k += F) {
    const int s0 = FORWARD ? begin + k : begin + share - F - k;
    if (!q.any_inside(s0, F)) continue;  // (frames outside the sequence change nothing)
    typename C::Raw raw[F][3];
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int t = q.frame_inside(s0 + j);
      const __amdgpu_buffer_rsrc_t row = X.at(X.of(t));
      raw[j][0] = C::C::load(row, FORWARD ? q.at[0] : q.at[3]);
      raw[j][1] = FORWARD ? C::C::load(row, q.at[1]) : C::C::load(DY.at(DY.of(t)), q.at[0]);
      raw[j][2] = C::C::load(row, q.at[2]);
    }
    auto add = [&](auto all) {
#pragma unroll
      for (int l = 0; l < F; ++l) {
        const int j = FORWARD ? l : F - 1 - l;
        float p[VEC], r[VEC], f[VEC];
        C::C::get(raw[j][0], p);
        C::C::get(raw[j][1], r);
        C::C::get(raw[j][2], f);
        const bool in = all || q.inside(s0 + j);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float fv = in ? Gate<AT>::sigmoid(f[v]) : 1.f;
          const float add = FORWARD ? Gate<AT>::sigmoid(r[v]) * Gate<AT>::tanh(p[v]) : r[v] * Gate<AT>::sigmoid(p[v]);
          run.a[v] *= fv;
          run.s[v] = FORWARD ? __builtin_fmaf(fv, run.s[v], in ? add : 0.f) : fv * (run.s[v] + (in ? add : 0.f));
        }
      }
    };
    if (q.all_inside(s0, F))
      add(std::true_type());
    else
      add(std::false_type());
  }
  handed[wave][q.lane] = run;
  __syncthreads();
  if (wave > 0) return;
  Run<VEC> all = Run<VEC>::none();
#pragma unroll
  for (int j = 0; j < W; ++j) all.then(handed[FORWARD ? j : W - 1 - j][q.lane]);
  ((Run<VEC>*)a.runs)[((size_t)segment * a.chains + chain) * 64 + q.lane] = all;
}

}  // namespace rtn
