// Host side of librtn_sequence_ops.so: argument checks and launches (include/rtn_sequence_ops.h).
#include "../../include/rtn_sequence_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "dropout_kernel.h"
#include "gated_recurrence_kernels.h"
#include "host_common.h"
#include "token_scores_kernels.h"

namespace rtn {
namespace {

// ---- gated recurrence ---------------------------------------------------------------------------------------------
// Frames that a wavefront holds at once, forward, with twice as many channels, and in the gradient: as many as leave 16 wavefronts their registers.
constexpr int kForwardFrames = 8, kWideFrames = 4, kGradientFrames = 4;

constexpr int64_t kMaxFrames = 1 << 30, kMaxChannels = 1 << 26;  // (steps are 32-bit numbers, and so is a place in a row, in bytes)

struct RecurrencePlan {
  int vec, waves, strips, segments;
  bool wide;
  int64_t chains, segment;
};
// Channels of a lane: what a word of 32 bits holds, pieces of 256 bytes for a wavefront.  In bf16 one, where two would leave half the lanes without any, or where that makes
// the most workgroups that run at once: each then has half the gates to compute (us, two / one: T=642 89 rows of n=64 forward 31.4 / 23.2, gradient 39.0 / 30.2; T=1000 n=512 32 rows
// 50.5 / 40.8 and 71.4 / 71.1, 16 rows 29.4 / 35.9 and 42.5 / 50.4; T=300 n=1024 10 rows 17.2 / 13.8 and 19.1 / 18.2, 20 rows 19.5 / 20.5 and 29.4 / 36.8).
// Forward, twice as many where that makes half as many workgroups that still fill the
// device (they read faster, 4.9 instead of 4.5 TB/s, but rounds that are not full cost more).  us, narrow / wide: T=500 n=1024 bf16 36 rows 56.9 / 52.4, 64 rows 72.7 / 67.7,
// 80 rows 94 / 105, 112 rows 128 / 121, 160 rows 170 / 179, 192 rows 208 / 194; T=300 n=512 float32 64 rows 47.3 / 42.6; T=64 64 rows of n=2048 bf16 18.2 / 19.1.
// (The gradient: 64 rows 130 / 128, with ragged lengths 117 / 129; 128 rows 243 / 227, 230 / 237.  It stays narrow.)
// Wavefronts: as few as take all frames at once, but no more than give every compute unit the 16 that it has registers for: 16 where all chains run at once so, else
// 8.  (us, 16 / 8: T=300 40 rows of n=512 float32 41.9 / 34.2; T=64 64 rows of n=2048 bf16 forward 23.5 / 18.5, gradient 33.4 / 28.6.  8 / 4 with 2048 chains
// and more: T=500 256 rows of n=1024 bf16 270 / 282 and 473 / 482, T=200 500 rows of n=512 float32 221 / 210 and 381 / 384.)
// Segments: as many as the time estimate is least for, in turns of W F frames: a workgroup takes its turns one after the other and half of one to start, 256 run
// at once; more than one segment costs the pre-pass, whose bytes are 0.6 (gradient 0.33) of the others, and a launch of 1.5.  Measured (us, one segment / these):
// T=4000 1 row of n=1024 bf16 forward 164 / 19, gradient 251 / 24; T=333 11 rows of n=1001 bf16 gradient 31.5 / 27.9; T=1000 32 rows of n=512 bf16 gradient 91 / 76.
RecurrencePlan recurrence_plan(int64_t T, int32_t B, int32_t n, int32_t dtype, bool gradient) {
  RecurrencePlan p;
  const int64_t of_one = (int64_t)((n + 63) / 64) * B;
  p.vec = dtype == RTN_DTYPE_BF16 && n > 64 && (of_one <= 128 || of_one > 256) ? 2 : 1;
  p.strips = (n + 64 * p.vec - 1) / (64 * p.vec);
  const int64_t half = (int64_t)p.strips / 2 * B, full_rounds = (half + 255) / 256 * 256;
  p.wide = !gradient && p.strips % 2 == 0 && T > 64 && half > 128 && (half <= 256 || 8 * half >= 7 * full_rounds);
  if (p.wide) p.vec *= 2, p.strips /= 2;
  p.chains = (int64_t)p.strips * B;
  const int frames = gradient ? kGradientFrames : (p.wide ? kWideFrames : kForwardFrames), most = p.chains > 256 ? 8 : 16;
  p.waves = 1;
  for (int w : {4, 8, 16})
    if (p.waves * frames < T && w <= most) p.waves = w;
  const int64_t turn = (int64_t)p.waves * frames, turns = std::max<int64_t>(1, (T + turn - 1) / turn);
  int64_t segments = 1;
  if (p.waves == 16 && !p.wide && p.chains <= 256) {
    auto estimate = [&](int64_t k) { return (double)((p.chains * k + 255) / 256) * ((turns + k - 1) / k + 0.5); };
    double least = estimate(1);
    for (int64_t k = 2; k <= std::min<int64_t>(turns, 512 / p.chains); ++k) {
      const double t = estimate(k) * (gradient ? 1.33 : 1.6) + 1.5;
      if (t < least) least = t, segments = k;
    }
  }
  const int64_t each = (turns + segments - 1) / segments;
  p.segment = each * turn;
  p.segments = (int)((turns + each - 1) / each);
  return p;
}
size_t recurrence_runs_bytes(const RecurrencePlan& p) { return p.segments > 1 ? (size_t)p.segments * (size_t)p.chains * 64 * p.vec * 8 : 0; }

// Whether no two strips of a row share a cache line of 128 bytes, in any of the arrays.
bool strips_apart(const RecurrencePlan& p, int B, int n, int dtype, std::initializer_list<const void*> arrays, std::initializer_list<int64_t> pitches) {
  const int64_t e = size_of(dtype);
  bool apart = n * e % 128 == 0;
  for (const void* q : arrays) apart = apart && aligned(q, 128);
  for (int64_t ld : pitches) apart = apart && ld * e % 128 == 0;
  return apart || p.chains == B;  // (or there is one strip to a row)
}

// Calls f with a value of the element type and the number of channels per lane and of wavefronts as types.
template <int N>
using Count = std::integral_constant<int, N>;
template <typename F>
void with_recurrence(int dtype, const RecurrencePlan& p, F f) {
  auto waves = [&](auto type, auto vec) {
    if (p.waves == 1)
      f(type, vec, Count<1>());
    else if (p.waves == 4)
      f(type, vec, Count<4>());
    else if (p.waves == 8)
      f(type, vec, Count<8>());
    else
      f(type, vec, Count<16>());
  };
  if (dtype == RTN_DTYPE_F32)
    waves(0.f, Count<1>());
  else if (p.vec == 2)
    waves((__bf16)0.f, Count<2>());
  else
    waves((__bf16)0.f, Count<1>());
}
// ... of a wide plan (more frames than one turn, so 8 or 16 wavefronts).
template <typename F>
void with_wide_recurrence(int dtype, const RecurrencePlan& p, F f) {
  auto waves = [&](auto type, auto vec) {
    if (p.waves == 8)
      f(type, vec, Count<8>());
    else
      f(type, vec, Count<16>());
  };
  if (dtype == RTN_DTYPE_F32)
    waves(0.f, Count<2>());
  else
    waves((__bf16)0.f, Count<4>());
}

// The checks that both directions share; `ld` is set where it was left out.
int recurrence_check(const char* what, const void* X, int64_t* ldX, const float* c0, const int64_t* lens, int64_t T, int32_t B, int32_t n, int32_t dtype, int32_t direction) {
  if (T < 0 || B < 0 || n < 0 || T > kMaxFrames || n > kMaxChannels) return fail(RTN_ERR_SHAPE, "%s: T=%lld B=%d n=%d", what, (long long)T, B, n);
  if (!known(dtype)) return fail(RTN_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (direction != 1 && direction != -1) return fail(RTN_ERR_RANGE, "%s: direction must be 1 or -1, got %d", what, direction);
  if (!*ldX) *ldX = 4 * (int64_t)n;
  if (*ldX < 4 * (int64_t)n) return fail(RTN_ERR_SHAPE, "%s: rows of X are %lld elements apart, but have %lld", what, (long long)*ldX, 4ll * n);
  if (T && B && n && !X) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  if (!aligned(X, size_of(dtype)) || !aligned(c0, 4) || !aligned(lens, 8)) return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  return RTN_OK;
}

}  // namespace
}  // namespace rtn

using namespace rtn;

extern "C" {

int rtn_sequence_ops_abi_version(void) { return 1; }
const char* rtn_sequence_last_error(void) { return g_last_error.c_str(); }

size_t rtn_gated_recurrence_saved_bytes(int64_t T, int32_t B, int32_t n, int32_t) {
  return T <= 0 || B <= 0 || n <= 0 ? 0 : (size_t)((T + kSavedFrames - 1) / kSavedFrames) * (size_t)B * (size_t)n * 4;
}
size_t rtn_gated_recurrence_fwd_workspace_bytes(int64_t T, int32_t B, int32_t n, int32_t dtype) {
  return T <= 0 || B <= 0 || n <= 0 ? 0 : recurrence_runs_bytes(recurrence_plan(T, B, n, dtype, false));
}
size_t rtn_gated_recurrence_bwd_workspace_bytes(int64_t T, int32_t B, int32_t n, int32_t dtype) {
  return T <= 0 || B <= 0 || n <= 0 ? 0 : recurrence_runs_bytes(recurrence_plan(T, B, n, dtype, true));
}

int rtn_gated_recurrence_fwd(const void* X, int64_t ldX, const float* c0, const int64_t* lens, void* Y, float* cN, void* saved, int64_t T, int32_t B, int32_t n,
                             int32_t dtype, int32_t direction, void* workspace, size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const int rc = recurrence_check("gated recurrence", X, &ldX, c0, lens, T, B, n, dtype, direction);
  if (rc != RTN_OK) return rc;
  if (B == 0 || n == 0) return RTN_OK;
  if ((T && !Y) || !cN) return fail(RTN_ERR_ARG, "gated recurrence: null pointer");
  if (!aligned(Y, size_of(dtype)) || !aligned(cN, 4) || !aligned(saved, 16)) return fail(RTN_ERR_ARG, "gated recurrence: misaligned pointer");
  const RecurrencePlan p = recurrence_plan(T, B, n, dtype, false);
  const size_t need = recurrence_runs_bytes(p);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "gated recurrence: workspace of %zu bytes needed", need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "gated recurrence: workspace must be 16-byte aligned");
  if (p.chains * p.segments > max_blocks(64 * p.waves)) return fail(RTN_ERR_SHAPE, "gated recurrence: B=%d n=%d are too many channels for one call", B, n);
  const int apart = strips_apart(p, B, n, dtype, {X, Y}, {ldX, n});
  const RecurrenceArgs a{X, ldX, c0, lens, Y, cN, (float*)saved, nullptr, 0, nullptr, nullptr, nullptr, T, B, n, direction < 0, p.strips, (unsigned)p.chains, p.segment, p.segments, apart, (float*)workspace};
  const hipStream_t stream = (hipStream_t)hip_stream;
  const dim3 grid((unsigned)(p.chains * p.segments));
  if (p.wide)
    with_wide_recurrence(dtype, p, [&](auto type, auto vec, auto waves) {
      constexpr int W = decltype(waves)::value;
      hipLaunchKernelGGL((k_recurrence_fwd<decltype(type), decltype(vec)::value, kWideFrames, W>), grid, dim3(64 * W), 0, stream, a);
    });
  else
    with_recurrence(dtype, p, [&](auto type, auto vec, auto waves) {
      typedef decltype(type) AT;
      constexpr int VEC = decltype(vec)::value, W = decltype(waves)::value;
      if constexpr (W == 16)
        if (p.segments > 1)
          hipLaunchKernelGGL((k_recurrence_runs<AT, VEC, kForwardFrames, W, true>), dim3((unsigned)(p.chains * (p.segments - 1))), dim3(64 * W), 0, stream, a);
      hipLaunchKernelGGL((k_recurrence_fwd<AT, VEC, kForwardFrames, W>), grid, dim3(64 * W), 0, stream, a);
    });
  return launched("gated recurrence");
}

int rtn_gated_recurrence_bwd(const void* X, int64_t ldX, const float* c0, const int64_t* lens, const void* saved, const void* DY, int64_t ldDY, const float* DcN, void* DX,
                             float* Dc0, int64_t T, int32_t B, int32_t n, int32_t dtype, int32_t direction, void* workspace, size_t workspace_bytes,
                             void* hip_stream) {
  g_last_error.clear();
  const int rc = recurrence_check("gated recurrence gradient", X, &ldX, c0, lens, T, B, n, dtype, direction);
  if (rc != RTN_OK) return rc;
  if (B == 0 || n == 0) return RTN_OK;
  if (!ldDY) ldDY = n;
  if (ldDY < n) return fail(RTN_ERR_SHAPE, "gated recurrence gradient: rows of DY are %lld elements apart, but have %d", (long long)ldDY, n);
  if ((T && (!DX || !DY || !saved)) || !Dc0) return fail(RTN_ERR_ARG, "gated recurrence gradient: null pointer");
  if (!aligned(DY, size_of(dtype)) || !aligned(DX, size_of(dtype)) || !aligned(Dc0, 4) || !aligned(DcN, 4) || !aligned(saved, 16))
    return fail(RTN_ERR_ARG, "gated recurrence gradient: misaligned pointer");
  const RecurrencePlan p = recurrence_plan(T, B, n, dtype, true);
  const size_t need = recurrence_runs_bytes(p);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "gated recurrence gradient: workspace of %zu bytes needed", need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "gated recurrence gradient: workspace must be 16-byte aligned");
  if (p.chains * p.segments > max_blocks(64 * p.waves)) return fail(RTN_ERR_SHAPE, "gated recurrence gradient: B=%d n=%d are too many channels for one call", B, n);
  const int apart = strips_apart(p, B, n, dtype, {X, DY, DX}, {ldX, ldDY, 4 * (int64_t)n});
  const RecurrenceArgs a{X, ldX, c0, lens, nullptr, nullptr, (float*)saved, DY, ldDY, DcN, DX, Dc0, T, B, n, direction < 0, p.strips, (unsigned)p.chains, p.segment, p.segments, apart, (float*)workspace};
  with_recurrence(dtype, p, [&](auto type, auto vec, auto waves) {
    typedef decltype(type) AT;
    constexpr int VEC = decltype(vec)::value, W = decltype(waves)::value;
    const hipStream_t stream = (hipStream_t)hip_stream;
    if constexpr (W == 16)
      if (p.segments > 1)
        hipLaunchKernelGGL((k_recurrence_runs<AT, VEC, kGradientFrames, W, false>), dim3((unsigned)(p.chains * (p.segments - 1))), dim3(64 * W), 0, stream, a);
    hipLaunchKernelGGL((k_recurrence_bwd<AT, VEC, kGradientFrames, W>), dim3((unsigned)(p.chains * p.segments)), dim3(64 * W), 0, stream, a);
  });
  return launched("gated recurrence gradient");
}

int rtn_dropout(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t times, int64_t rows, int64_t width, int32_t dtype, int32_t threshold,
                uint64_t seed, uint64_t offset, const int64_t* offset_ptr, int32_t same_over_time, void* hip_stream) {
  g_last_error.clear();
  if (times < 0 || rows < 0 || width < 0) return fail(RTN_ERR_SHAPE, "dropout: [%lld,%lld,%lld]", (long long)times, (long long)rows, (long long)width);
  if (!known(dtype)) return fail(RTN_ERR_ARG, "dropout: unknown dtype %d", dtype);
  if (threshold < 0 || threshold > 65536) return fail(RTN_ERR_RANGE, "dropout: threshold %d is not in 0..65536", threshold);
  if (!ldx) ldx = width;
  if (!ldr) ldr = width;
  if (ldx < width || ldr < width) return fail(RTN_ERR_SHAPE, "dropout: rows are %lld and %lld elements apart, but have %lld", (long long)ldx, (long long)ldr, (long long)width);
  if (!times || !rows || !width) return RTN_OK;
  if (!x || !y) return fail(RTN_ERR_ARG, "dropout: null pointer");
  const int e = size_of(dtype);
  if (!aligned(x, e) || !aligned(y, e) || !aligned(residual, e) || !aligned(offset_ptr, 8)) return fail(RTN_ERR_ARG, "dropout: misaligned pointer");
  const float scale = threshold == 65536 ? 0.f : 65536.f / (float)(65536 - threshold);
  if (!same_over_time) {
    if (rows > INT64_MAX / times) return fail(RTN_ERR_SHAPE, "dropout: [%lld,%lld,%lld] is too large for one call", (long long)times, (long long)rows, (long long)width);
    rows *= times, times = 1;
  }
  const int64_t count = rows * width, groups = (count + 7) / 8;
  const bool flat = (rows == 1 && times == 1) || (ldx == width && (!residual || ldr == width));
  const int64_t blocks = flat ? (groups * times + 511) / 512 : (groups + 255) / 256;
  if (blocks > max_blocks(256)) return fail(RTN_ERR_SHAPE, "dropout: [%lld,%lld,%lld] is too large for one call", (long long)times, (long long)rows, (long long)width);
  const DropoutArgs a{x, residual, y, ldx, ldr, times, rows, width, count, (unsigned)threshold, scale, (unsigned)seed, (unsigned)(seed >> 32), offset, offset_ptr};
  with_type(dtype, [&](auto type) {
    typedef decltype(type) AT;
    with_bool(residual != nullptr, [&](auto add) {
      constexpr bool ADD = decltype(add)::value;
      const hipStream_t stream = (hipStream_t)hip_stream;
      if (!flat)
        hipLaunchKernelGGL((k_dropout_rows<AT, ADD>), dim3((unsigned)blocks, (unsigned)std::min<int64_t>(times, 65535)), dim3(256), 0, stream, a);
      else if (times > 1)
        hipLaunchKernelGGL((k_dropout<AT, ADD, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((k_dropout<AT, ADD, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    });
  });
  return launched("dropout");
}

// ---- scores of tokens ---------------------------------------------------------------------------------------------
static int scores_check(const char* what, const void* logits, int64_t* ld, const int64_t* targets, int64_t rows, int64_t V, int32_t dtype) {
  if (rows < 0 || V < 0 || V > kMaxTokens) return fail(RTN_ERR_SHAPE, "%s: %lld rows of %lld logits (at most %lld)", what, (long long)rows, (long long)V, (long long)kMaxTokens);
  if (rows > kMaxRows) return fail(RTN_ERR_SHAPE, "%s: %lld rows are too many for one call", what, (long long)rows);
  if (!known(dtype)) return fail(RTN_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (!*ld) *ld = V;
  if (*ld < V) return fail(RTN_ERR_SHAPE, "%s: rows are %lld elements apart, but have %lld", what, (long long)*ld, (long long)V);
  if (rows && V == 0) return fail(RTN_ERR_SHAPE, "%s: rows without a logit", what);
  if (rows && !logits) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  if (!aligned(logits, size_of(dtype)) || !aligned(targets, 8)) return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  return RTN_OK;
}

// Pieces of a row: where alternatives are wanted, as many as it takes for 16 wavefronts to hold a piece in registers, or, where that are several and few rows leave
// most of the device idle, for 8 wavefronts with half as many logits each (us, the former / the latter, 20 alternatives of float32: one row of 131072 10.4 / 8.6, 12 rows of
// 131072 11.5 / 10.3, 40 rows of 131072 13.8 / 14.8, one row of 10^6 11.8 / 24.3).  Else one, but where rows are few as many as in the first case.
constexpr int kSmallSegment = 8 * 64 * 16;
static int64_t scores_splits(int64_t rows, int64_t V, int32_t top_k) {
  const int64_t pieces = (V + kMaxSegment - 1) / kMaxSegment, small = (V + kSmallSegment - 1) / kSmallSegment;
  if (top_k > 0 && pieces > 1 && small <= 64 && rows * small <= 256) return small;
  return top_k > 0 || rows < 256 ? pieces : 1;
}

size_t rtn_token_log_probs_workspace_bytes(int64_t rows, int64_t V, int32_t, int32_t top_k) {
  if (rows <= 0 || V <= 0 || top_k < 0) return 0;
  const int64_t splits = scores_splits(rows, V, top_k);
  return splits == 1 ? 0 : (size_t)rows * (size_t)splits * (16 + 8 * (size_t)top_k);
}

int rtn_token_log_probs_fwd(const void* logits, int64_t ld, const int64_t* targets, int64_t rows, int64_t V, int32_t dtype, int32_t top_k, float* log_prob, float* norm,
                            float* entropy, float* top_log_prob, int64_t* top_ids, void* workspace, size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const int rc = scores_check("token log probabilities", logits, &ld, targets, rows, V, dtype);
  if (rc != RTN_OK) return rc;
  if (top_k < 0 || top_k > kMaxAlternatives || (rows && top_k > V))
    return fail(RTN_ERR_RANGE, "token log probabilities: %d alternatives of %lld tokens (at most %d)", top_k, (long long)V, kMaxAlternatives);
  if (rows == 0) return RTN_OK;
  if (log_prob && !targets) return fail(RTN_ERR_ARG, "token log probabilities: no targets");
  if (top_k && (!top_log_prob || !top_ids)) return fail(RTN_ERR_ARG, "token log probabilities: null pointer");
  if (!aligned(log_prob, 4) || !aligned(norm, 8) || !aligned(entropy, 4) || !aligned(top_log_prob, 4) || !aligned(top_ids, 8))
    return fail(RTN_ERR_ARG, "token log probabilities: misaligned pointer");
  const int64_t splits = scores_splits(rows, V, top_k), segment = splits == 1 ? V : ((V + splits - 1) / splits + 7) / 8 * 8;
  const size_t need = rtn_token_log_probs_workspace_bytes(rows, V, dtype, top_k);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "token log probabilities: workspace of %zu bytes needed", need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "token log probabilities: workspace must be 16-byte aligned");
  const ScoresArgs a{logits, ld,      targets, rows,    (int)V,      top_k,           log_prob,
                     norm,   entropy, top_log_prob, top_ids, nullptr, nullptr, nullptr,
                     (int)splits, (int)segment, (float*)workspace, (unsigned long long*)((char*)workspace + (size_t)rows * (size_t)splits * 16)};
  const int64_t one = rows * splits, four = (rows + 3) / 4, sixteen = (rows + 15) / 16;
  bool fits = true;
  auto launch = [&](void (*kernel)(ScoresArgs), int64_t blocks, int threads) {
    if (blocks > max_blocks(threads))
      fits = false;
    else
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), 0, (hipStream_t)hip_stream, a);
  };
  with_type(dtype, [&](auto type) {
    typedef decltype(type) AT;
    // Short rows 16 at a time, but not for many alternatives, of which 16 lanes' maxima tell too little (us, 2000 rows of 96 bf16, one wavefront per row / this: sums 3.5 / 2.7, 5 alternatives 4.6 / 4.1,
    // 16 alternatives 7.1 / 15.0; 70000 rows 25 / 6.7, 41 / 13.5, 56 / 86).
    if (V >= 8 && V <= 256 && top_k <= 8) {
      if (V <= 128)
        launch(k_token_scores_short<AT, 8>, sixteen, 256);
      else
        launch(k_token_scores_short<AT, 16>, sixteen, 256);
      return;
    }
    if (top_k > 0) {
      // As few wavefronts as hold a piece, but where rows are few (up to 512: two workgroups a compute unit, which leave most of it idle), more of them with less each (us, with 5 alternatives: 64 rows of 500 bf16 a wavefront each 6.5, four
      // 5.1, 1024 rows 5.4 / 6.2; 64 rows of 8000 float32 four 5.8, eight 5.1, 2048 rows 16.9 / 17.3; 3000 rows of 4000 bf16 four 12.3, eight 18.0).  Lanes hold no
      // more than it takes (3000 rows of 20000 bf16 32 logits 46.7, 24 41.5; 5000 of 10007 42.5 / 38.2).
      // Many of up to 2048 logits (above 1024 rows: four wavefronts a compute unit and more, if a row has only one) take one wavefront, without barriers (29000 rows of 1000 bf16 four 61, one 27, of 2000 64 and 38; 700 rows of 2000 5.2 and 5.7).
      const bool few = rows <= 512, many = rows > 1024;
      if (segment <= 64 || (segment <= 512 && !few))
        launch(k_token_scores_top<AT, 1, 8>, four, 256);
      else if (segment <= 1024 && many)
        launch(k_token_scores_top<AT, 1, 16>, four, 256);
      else if (segment <= 2048 && many)
        launch(k_token_scores_top<AT, 1, 32>, four, 256);
      else if (segment <= 2048)
        launch(k_token_scores_top<AT, 4, 8>, one, 256);
      else if (segment <= 4096)
        launch(k_token_scores_top<AT, 4, 16>, one, 256);
      else if (segment <= 8192 && few)
        launch(k_token_scores_top<AT, 8, 16>, one, 512);
      else if (segment <= 6144)
        launch(k_token_scores_top<AT, 4, 24>, one, 256);
      else if (segment <= 8192)
        launch(k_token_scores_top<AT, 4, 32>, one, 256);
      else if (segment <= 12288)
        launch(k_token_scores_top<AT, 8, 24>, one, 512);
      else if (segment <= 16384)
        launch(k_token_scores_top<AT, 8, 32>, one, 512);
      else if (segment <= 24576)
        launch(k_token_scores_top<AT, 16, 24>, one, 1024);
      else
        launch(k_token_scores_top<AT, 16, 32>, one, 1024);
    } else {
      with_bool(entropy != nullptr, [&](auto with_entropy) {
        constexpr bool ENTROPY = decltype(with_entropy)::value;
        // (us of bf16 rows, one wavefront / four: 9000 of 1500 9.4 / 11.5, 9000 of 6000 25.0 / 21.5; four / sixteen: 100 of 32000 7.1 / 5.8, 4096 of 16000 30.2 / 35.5)
        if (segment <= 1536)
          launch(k_token_scores<AT, 1, ENTROPY>, four, 256);
        else if (rows >= 256 || segment <= 8192)
          launch(k_token_scores<AT, 4, ENTROPY>, one, 256);
        else
          launch(k_token_scores<AT, 16, ENTROPY>, one, 1024);
      });
    }
    if (splits > 1 && fits) {
      // (16 lanes per alternative, but no more wavefronts than are there at once)
      const int threads = rows > 512 ? 256 : (int)std::clamp<int64_t>((16 * splits * top_k + 63) / 64 * 64, 256, 1024);
      launch(k_token_scores_join<AT>, rows, threads);
    }
  });
  if (!fits) return fail(RTN_ERR_SHAPE, "token log probabilities: %lld rows of %lld are too many for one call", (long long)rows, (long long)V);
  return launched("token log probabilities");
}

int rtn_token_log_probs_bwd(const void* logits, int64_t ld, const int64_t* targets, const float* norm, const float* entropy, const float* d_log_prob, const float* d_entropy,
                            void* D, int64_t rows, int64_t V, int32_t dtype, void* hip_stream) {
  g_last_error.clear();
  const int rc = scores_check("token log probabilities gradient", logits, &ld, targets, rows, V, dtype);
  if (rc != RTN_OK) return rc;
  if (rows == 0) return RTN_OK;
  if (!D || !norm || (d_entropy && !entropy) || (d_log_prob && !targets)) return fail(RTN_ERR_ARG, "token log probabilities gradient: null pointer");
  if (!aligned(D, size_of(dtype)) || !aligned(norm, 8) || !aligned(entropy, 4) || !aligned(d_log_prob, 4) || !aligned(d_entropy, 4))
    return fail(RTN_ERR_ARG, "token log probabilities gradient: misaligned pointer");
  const int64_t pieces = (V + kBwdPiece - 1) / kBwdPiece;
  const int64_t blocks = V <= 256 ? (rows + 15) / 16 : (V <= 2048 ? (rows + 3) / 4 : rows * pieces);
  if (blocks > max_blocks(256)) return fail(RTN_ERR_SHAPE, "token log probabilities gradient: %lld rows of %lld are too many for one call", (long long)rows, (long long)V);
  const ScoresArgs a{logits,  ld,      targets, rows,       (int)V,    0, nullptr,     (float*)norm, (float*)entropy,
                     nullptr, nullptr, d_log_prob, d_entropy, D, (int)pieces, 0, nullptr, nullptr};
  with_type(dtype, [&](auto type) {
    typedef decltype(type) AT;
    // (us of bf16 rows, a wavefront per row / 16 lanes: 70000 of 96 21.4 / 9.0, 10000 of 256 6.2 / 5.3, 37 of 256 3.4 / 3.6; a wavefront / a workgroup per piece: 9000 of 500
    // 8.6 / 13.5, of 2000 18.4 / 19.7, of 5000 46.6 / 37.7)
    if (V <= 256)
      hipLaunchKernelGGL((k_token_scores_bwd<AT, 16>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)hip_stream, a);
    else if (V <= 2048)
      hipLaunchKernelGGL((k_token_scores_bwd<AT, 64>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)hip_stream, a);
    else
      hipLaunchKernelGGL((k_token_scores_bwd<AT, 256>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)hip_stream, a);
  });
  return launched("token log probabilities gradient");
}

}  // extern "C"
