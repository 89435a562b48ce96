// Host side of librtn_model_ops.so: argument checks and launches (include/rtn_model_ops.h).
#include "../../include/rtn_model_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <utility>

#include "beam_kernels.h"
#include "delta_rule_kernels.h"
#include "embedding_kernels.h"
#include "host_common.h"

namespace rtn {
namespace {

constexpr int64_t kMaxFrames = 1 << 30;  // (as of the gated recurrence)
constexpr int kMaxKeyDim = 128, kMaxValueDim = 65536;

// ---- gated delta rule -----------------------------------------------------------------------------------------------
struct DeltaSizes {
  int64_t T;
  int32_t B, key_heads, heads, dk, dv, dtype;
};
bool nothing(const DeltaSizes& z) { return z.B == 0 || z.heads == 0; }
bool valid(const DeltaSizes& z) {
  return z.T >= 0 && z.T <= kMaxFrames && z.B >= 0 && z.key_heads >= 0 && z.heads >= 0 && z.dk >= 1 && z.dk <= kMaxKeyDim && z.dv >= 1 && z.dv <= kMaxValueDim && known(z.dtype);
}
// Calls of at most these frames that no gradient follows go frame by frame.  (12 sequences of 8 heads of 128 x 128 in bf16, frame by frame and in chunks: 1 frame 5.9 and 33 us, 16 frames 25.1 and
// 30.7, 24 frames 35 and 31.5; 16 frames of one sequence 23.7 and 29.3, of 64 52 and 54.)
constexpr int kStepFrames = 16;
int delta_frames(const DeltaSizes& z) { return z.dtype == RTN_DTYPE_BF16 ? DeltaChunk<__bf16>::kFrames : DeltaChunk<float>::kFrames; }
int64_t delta_chunks(const DeltaSizes& z) { return (z.T + delta_frames(z) - 1) / delta_frames(z); }
size_t delta_all_chunks(const DeltaSizes& z) { return (size_t)z.B * (size_t)z.heads * (size_t)delta_chunks(z); }
// Numbers of float32 in the sections of what the gradient wants to know, and of its workspace.
size_t delta_records(const DeltaSizes& z) { return delta_all_chunks(z) * (size_t)delta_record(delta_frames(z)); }
int delta_key_width(const DeltaSizes& z) { return z.dk <= 32 ? 32 : (z.dk <= 64 ? 64 : 128); }
size_t delta_states(const DeltaSizes& z) { return delta_all_chunks(z) * (size_t)delta_key_width(z) * (size_t)z.dv; }
size_t delta_writes(const DeltaSizes& z) { return delta_all_chunks(z) * (size_t)delta_frames(z) * (size_t)z.dv; }
size_t delta_shared(const DeltaSizes& z) { return z.heads == z.key_heads ? 0 : (size_t)z.T * (size_t)z.B * (size_t)z.heads * (size_t)z.dk; }

// Calls f with a value of the element type and the keys' width in LDS as a type.
template <int N>
using Count = std::integral_constant<int, N>;
template <typename F>
void with_delta(const DeltaSizes& z, F f) {
  with_type(z.dtype, [&](auto type) {
    if (z.dk <= 32)
      f(type, Count<32>());
    else if (z.dk <= 64)
      f(type, Count<64>());
    else
      f(type, Count<128>());
  });
}
// Wavefronts of a workgroup that goes through a head's chunks, with 16 columns of the state each.  Four take three quarters of the time that eight take, for half the columns: T=1000, heads of
// 128 x 128 in bf16, four and eight: 128 heads (one round of workgroups, one) 147 and 191 us, with the gradient 553 and 640; 256 heads (two, one) 313 and 284, 1071 and 946.
int delta_waves(const DeltaSizes& z) {
  const int64_t lines = (int64_t)z.B * z.heads, four = (lines * ((z.dv + 63) / 64) + 255) / 256, eight = (lines * ((z.dv + 127) / 128) + 255) / 256;  // rounds of the device
  return 4 * eight < 3 * four ? 8 : 4;
}
int64_t delta_strips(const DeltaSizes& z) { return (z.dv + 16 * delta_waves(z) - 1) / (16 * delta_waves(z)); }
template <typename F>
void with_waves(const DeltaSizes& z, F f) {
  if (delta_waves(z) == 8)
    f(Count<8>());
  else
    f(Count<4>());
}
constexpr int kSegmentWaves = 4;
// Segments of the chunks, where sequences and heads are few: as many as a time estimate is least for, in which a chunk takes 1 (and 0.8 more in the first pass), a border 0.3, and both
// passes run in rounds of as many workgroups as there are compute units.  T=4000, one sequence of 8 heads of 128 x 128 in bf16: one segment 354 us, 4 166, 8 110, 16 (chosen) 96-100;
// T=8192, two of 8 heads of 64 x 128: 584, 265, 175, 181-185 (chosen), 32 196; T=1000, 16 of 8 of 128 x 128: one (chosen) 146, 4 274.  One segment or at least three; where eight wavefronts are taken half of the compute units
// have work, and the estimate never finds segments worth their second pass.
int64_t delta_segments(const DeltaSizes& z) {
  if (delta_waves(z) != kSegmentWaves) return 1;
  const int64_t chunks = delta_chunks(z), lines = (int64_t)z.B * z.heads, width = 16 * kSegmentWaves;
  const int64_t strips = delta_strips(z), strips_through = ((z.dv + 15) / 16 * 16 + delta_key_width(z) + width - 1) / width;
  auto rounds = [&](int64_t blocks) { return (double)((blocks + 255) / 256); };
  double least = rounds(lines * strips) * chunks;
  int64_t best = 1;
  for (int64_t some : {3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256}) {
    if (some > chunks / 2 || lines * strips * some > 1024) break;
    const int64_t per = (chunks + some - 1) / some, n = (chunks + per - 1) / per;
    const double t = per * (rounds(lines * strips * n) + 0.8 * rounds(lines * strips_through * (n - 1))) + 0.3 * n + 3;
    if (t < least) least = t, best = n;
  }
  return best;
}
size_t delta_borders(const DeltaSizes& z) { return (size_t)(delta_segments(z) - 1) * z.B * z.heads * delta_key_width(z) * z.dv; }
size_t delta_through(const DeltaSizes& z) { return (size_t)(delta_segments(z) - 1) * z.B * z.heads * 3 * delta_key_width(z) * delta_key_width(z) / 2; }

// Whether launches and offsets are within what 32 bits count; widest: elements of a frame of the widest tensor, with its pitch.
bool delta_fits(const DeltaSizes& z, int64_t widest) {
  const int64_t most = max_blocks(512) / std::max<int64_t>(1, (int64_t)z.B * z.heads);
  return delta_chunks(z) <= most && delta_strips(z) <= most && (!delta_shared(z) || delta_shared(z) / 256 < (size_t)max_blocks(256)) &&
         std::max(widest, (int64_t)z.heads * z.dv) <= kDeltaFrameBytes / size_of(z.dtype) / z.B;
}
int delta_check(const char* what, const DeltaSizes& z, int32_t direction) {
  if (z.T < 0 || z.B < 0 || z.key_heads < 0 || z.heads < 0 || z.T > kMaxFrames || z.dk < 1 || z.dk > kMaxKeyDim || z.dv < 1 || z.dv > kMaxValueDim)
    return fail(RTN_ERR_SHAPE, "%s: T=%lld B=%d key_heads=%d heads=%d dk=%d dv=%d (dk 1 to %d, dv 1 to %d)", what, (long long)z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, kMaxKeyDim,
                kMaxValueDim);
  if (z.key_heads ? z.heads % z.key_heads : z.heads) return fail(RTN_ERR_SHAPE, "%s: %d heads cannot share %d heads of queries and keys evenly", what, z.heads, z.key_heads);
  if (!known(z.dtype)) return fail(RTN_ERR_ARG, "%s: unknown dtype %d", what, z.dtype);
  if (direction != 1 && direction != -1) return fail(RTN_ERR_RANGE, "%s: direction must be 1 or -1, got %d", what, direction);
  return RTN_OK;
}
int pitch_check(const char* what, const char* name, int64_t* ld, int64_t width) {
  if (!*ld) *ld = width;
  return *ld < width ? fail(RTN_ERR_SHAPE, "%s: rows of %s are %lld elements apart, but have %lld", what, name, (long long)*ld, (long long)width) : RTN_OK;
}

}  // namespace
}  // namespace rtn

using namespace rtn;

extern "C" {

int rtn_model_ops_abi_version(void) { return 1; }
const char* rtn_model_ops_last_error(void) { return g_last_error.c_str(); }

size_t rtn_delta_rule_fwd_workspace_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype, int32_t keep) {
  const DeltaSizes z{T, B, key_heads, heads, dk, dv, dtype};
  if (!valid(z) || nothing(z) || (!keep && T <= kStepFrames)) return 0;
  return ((keep ? 0 : delta_records(z)) + delta_borders(z) + delta_through(z)) * 4;
}
size_t rtn_delta_rule_saved_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype) {
  const DeltaSizes z{T, B, key_heads, heads, dk, dv, dtype};
  return valid(z) && !nothing(z) ? (delta_records(z) + delta_through(z) + delta_states(z) + delta_writes(z)) * 4 : 0;
}
size_t rtn_delta_rule_bwd_workspace_bytes(int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype) {
  const DeltaSizes z{T, B, key_heads, heads, dk, dv, dtype};
  return valid(z) && !nothing(z) ? (delta_borders(z) + delta_states(z) + delta_writes(z) + 2 * delta_shared(z)) * 4 : 0;
}

int rtn_delta_rule_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* g, const float* beta, const float* s0,
                       const int64_t* lens, void* y, float* sN, void* saved, int64_t T, int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv,
                       int32_t dtype, float scale, int32_t direction, void* workspace, size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const char* what = "delta rule";
  const DeltaSizes z{T, B, key_heads, heads, dk, dv, dtype};
  int rc = delta_check(what, z, direction);
  if (rc == RTN_OK) rc = pitch_check(what, "q", &ldq, (int64_t)key_heads * dk);
  if (rc == RTN_OK) rc = pitch_check(what, "k", &ldk, (int64_t)key_heads * dk);
  if (rc == RTN_OK) rc = pitch_check(what, "v", &ldv, (int64_t)heads * dv);
  if (rc != RTN_OK) return rc;
  if (nothing(z)) return RTN_OK;
  if ((T && (!q || !k || !v || !g || !beta || !y)) || !sN) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  const int e = size_of(dtype);
  if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(y, e) || !aligned(g, 4) || !aligned(beta, 4) || !aligned(s0, 4) || !aligned(sN, 4) || !aligned(lens, 8) ||
      !aligned(saved, 16))
    return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  const DeltaArgs a{q, k, v, ldq, ldk, ldv, g, beta, s0, lens, y, sN, T, B, key_heads, heads, dk, dv, scale, direction < 0};
  const hipStream_t stream = (hipStream_t)hip_stream;
  if (!saved && T <= kStepFrames) {
    const int64_t blocks = (int64_t)B * heads * ((dv + 63) / 64);
    if (blocks > max_blocks(256)) return fail(RTN_ERR_SHAPE, "%s: B=%d heads=%d dv=%d are too many for one call", what, B, heads, dv);
    with_delta(z, [&](auto type, auto width) {
      hipLaunchKernelGGL((k_delta_steps<decltype(type), decltype(width)::value / 16>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    });
    return launched(what);
  }
  if (!delta_fits(z, std::max({ldq, ldk, ldv}))) return fail(RTN_ERR_SHAPE, "%s: T=%lld B=%d heads=%d dv=%d are too many for one call", what, (long long)T, B, heads, dv);
  const size_t need = rtn_delta_rule_fwd_workspace_bytes(T, B, key_heads, heads, dk, dv, dtype, saved != nullptr);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  DeltaChunkArgs c{};
  c.f = a, c.chunks = (int)delta_chunks(z);
  c.segments = (int)delta_segments(z), c.per = (int)((c.chunks + c.segments - 1) / c.segments);
  float* free = (float*)workspace;
  c.through = (__bf16*)free, free += delta_through(z);
  c.borders = free, free += delta_borders(z);
  c.records = (float*)(saved ? saved : free);
  if (saved) {
    c.through_t = (__bf16*)(c.records + delta_records(z));
    c.states = c.records + delta_records(z) + delta_through(z), c.writes = c.states + delta_states(z);
  }
  with_delta(z, [&](auto type, auto width) {
    typedef decltype(type) AT;
    constexpr int DK = decltype(width)::value;
    const dim3 heads_grid((unsigned)(B * heads * c.segments * delta_strips(z)));
    if (T) hipLaunchKernelGGL((k_delta_chunks<AT, DK>), dim3((unsigned)delta_all_chunks(z)), dim3(DeltaChunk<AT>::kFrames * 4), 0, stream, c);
    if (c.segments > 1) {
      const int64_t strips = ((dv + 15) / 16 * 16 + DK + 16 * kSegmentWaves - 1) / (16 * kSegmentWaves);
      hipLaunchKernelGGL((k_delta_forward<AT, DK, kSegmentWaves, kDeltaThrough>), dim3((unsigned)(B * heads * (c.segments - 1) * strips)), dim3(64 * kSegmentWaves), 0, stream, c);
      hipLaunchKernelGGL((k_delta_join<AT, DK, false>), dim3((unsigned)(B * heads * ((dv + 15) / 16))), dim3(DK * 4), 0, stream, c);
    }
    with_waves(z, [&](auto waves) {
      constexpr int W = decltype(waves)::value;
      if (saved)
        hipLaunchKernelGGL((k_delta_forward<AT, DK, W, kDeltaKeep>), heads_grid, dim3(64 * W), 0, stream, c);
      else
        hipLaunchKernelGGL((k_delta_forward<AT, DK, W, kDeltaPlain>), heads_grid, dim3(64 * W), 0, stream, c);
    });
  });
  return launched(what);
}

int rtn_delta_rule_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* g, const float* beta, const int64_t* lens,
                       const void* saved, const void* dy, int64_t lddy, const float* dsN, void* dq, void* dk_out, void* dv_out, float* dg, float* dbeta, float* ds0, int64_t T,
                       int32_t B, int32_t key_heads, int32_t heads, int32_t dk, int32_t dv, int32_t dtype, float scale, int32_t direction, void* workspace,
                       size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const char* what = "delta rule gradient";
  const DeltaSizes z{T, B, key_heads, heads, dk, dv, dtype};
  int rc = delta_check(what, z, direction);
  if (rc == RTN_OK) rc = pitch_check(what, "q", &ldq, (int64_t)key_heads * dk);
  if (rc == RTN_OK) rc = pitch_check(what, "k", &ldk, (int64_t)key_heads * dk);
  if (rc == RTN_OK) rc = pitch_check(what, "v", &ldv, (int64_t)heads * dv);
  if (rc == RTN_OK) rc = pitch_check(what, "dy", &lddy, (int64_t)heads * dv);
  if (rc != RTN_OK) return rc;
  if (nothing(z)) {  // (keys may be there without values: sums over no heads)
    if (!T || !B || !key_heads) return RTN_OK;
    if (!dq || !dk_out) return fail(RTN_ERR_ARG, "%s: null pointer", what);
    if (!aligned(dq, size_of(dtype)) || !aligned(dk_out, size_of(dtype))) return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
    if (T > max_blocks(256) * 256 / dk / B / key_heads) return fail(RTN_ERR_SHAPE, "%s: T=%lld B=%d key_heads=%d are too many for one call", what, (long long)T, B, key_heads);
    DeltaChunkArgs c{};
    c.f.T = T, c.f.B = B, c.f.key_heads = key_heads, c.f.dk = dk, c.dq = dq, c.dk = dk_out;
    with_type(dtype, [&](auto type) {
      hipLaunchKernelGGL(k_delta_shared<decltype(type)>, dim3((unsigned)((T * B * key_heads * (int64_t)dk + 255) / 256)), dim3(256), 0, (hipStream_t)hip_stream, c);
    });
    return launched(what);
  }
  if ((T && (!q || !k || !v || !g || !beta || !dy || !saved || !dq || !dk_out || !dv_out || !dg || !dbeta)) || !ds0) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  const int e = size_of(dtype);
  if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(dy, e) || !aligned(dq, e) || !aligned(dk_out, e) || !aligned(dv_out, e) || !aligned(g, 4) || !aligned(beta, 4) ||
      !aligned(dsN, 4) || !aligned(dg, 4) || !aligned(dbeta, 4) || !aligned(ds0, 4) || !aligned(lens, 8) || !aligned(saved, 16))
    return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  if (!delta_fits(z, std::max({ldq, ldk, ldv, lddy}))) return fail(RTN_ERR_SHAPE, "%s: T=%lld B=%d heads=%d dv=%d are too many for one call", what, (long long)T, B, heads, dv);
  const size_t need = rtn_delta_rule_bwd_workspace_bytes(T, B, key_heads, heads, dk, dv, dtype);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  DeltaChunkArgs c{};
  c.f = DeltaArgs{q, k, v, ldq, ldk, ldv, g, beta, nullptr, lens, nullptr, nullptr, T, B, key_heads, heads, dk, dv, scale, direction < 0};
  c.chunks = (int)delta_chunks(z);
  c.segments = (int)delta_segments(z), c.per = (int)((c.chunks + c.segments - 1) / c.segments);
  c.records = (float*)saved, c.through_t = (__bf16*)(c.records + delta_records(z));
  c.states = c.records + delta_records(z) + delta_through(z), c.writes = c.states + delta_states(z);
  c.dy = dy, c.lddy = lddy, c.dsN = dsN;
  c.borders = (float*)workspace;
  c.dstates = c.borders + delta_borders(z), c.dwrites = c.dstates + delta_states(z);
  if (delta_shared(z)) c.dq_each = c.dwrites + delta_writes(z), c.dk_each = c.dq_each + delta_shared(z);
  c.dq = dq, c.dk = dk_out, c.dv = dv_out, c.dg = dg, c.dbeta = dbeta, c.ds0 = ds0;
  with_delta(z, [&](auto type, auto width) {
    typedef decltype(type) AT;
    constexpr int DK = decltype(width)::value;
    const hipStream_t stream = (hipStream_t)hip_stream;
    if (c.segments > 1) {
      hipLaunchKernelGGL((k_delta_backward<AT, DK, kSegmentWaves, true>), dim3((unsigned)(B * heads * (c.segments - 1) * delta_strips(z))), dim3(64 * kSegmentWaves), 0, stream, c);
      hipLaunchKernelGGL((k_delta_join<AT, DK, true>), dim3((unsigned)(B * heads * ((dv + 15) / 16))), dim3(DK * 4), 0, stream, c);
    }
    with_waves(z, [&](auto waves) {
      constexpr int W = decltype(waves)::value;
      hipLaunchKernelGGL((k_delta_backward<AT, DK, W, false>), dim3((unsigned)(B * heads * c.segments * delta_strips(z))), dim3(64 * W), 0, stream, c);
    });
    if (T)
      with_bool(dv < 8, [&](auto narrow) {
        hipLaunchKernelGGL((k_delta_gradients<AT, DK, decltype(narrow)::value>), dim3((unsigned)delta_all_chunks(z)), dim3(DK * 4), 0, stream, c);
      });
    if (delta_shared(z)) {
      const int64_t items = T * B * key_heads * (int64_t)dk;
      hipLaunchKernelGGL(k_delta_shared<AT>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, c);
    }
  });
  return launched(what);
}

// ---- embedding ------------------------------------------------------------------------------------------------------
static int embedding_check(const char* what, const int64_t* tokens, const void* in, int64_t* ld, const void* out, int64_t rows, int64_t V, int64_t D, int32_t dtype) {
  if (rows < 0 || rows > kMaxRows || V < 0 || V > kMaxRows || D < 0) return fail(RTN_ERR_SHAPE, "%s: %lld rows of a table [%lld,%lld]", what, (long long)rows, (long long)V, (long long)D);
  if (!known(dtype)) return fail(RTN_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (const int rc = pitch_check(what, "the input", ld, D); rc != RTN_OK) return rc;
  const int e = size_of(dtype);
  if (!aligned(tokens, 8) || !aligned(in, e) || !aligned(out, e)) return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  return RTN_OK;
}

int rtn_embedding_fwd(const int64_t* tokens, const void* table, int64_t ld, void* y, int64_t rows, int64_t V, int64_t D, int32_t dtype, float scale, void* hip_stream) {
  g_last_error.clear();
  const char* what = "embedding";
  const int rc = embedding_check(what, tokens, table, &ld, y, rows, V, D, dtype);
  if (rc != RTN_OK) return rc;
  if (!rows || !D) return RTN_OK;
  if (!tokens || !y || (V && !table)) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  const EmbeddingArgs a{tokens, table, ld, y, rows, V, D, scale, nullptr, nullptr};
  const int64_t groups = (D + 7) / 8;
  if (groups > max_blocks(256) * 256 / rows) return fail(RTN_ERR_SHAPE, "%s: %lld rows of %lld are too many for one call", what, (long long)rows, (long long)D);
  with_type(dtype, [&](auto type) {
    hipLaunchKernelGGL(k_embedding<decltype(type)>, dim3((unsigned)((rows * groups + 255) / 256)), dim3(256), 0, (hipStream_t)hip_stream, a);
  });
  return launched(what);
}

// Workspace of the gradient: the sorted rows and their tokens, twice and counts of digits where there is more than one pass of sorting; the sums of runs over several pieces.
struct EmbeddingPlan {
  int64_t pieces, strips, blocks, pitch;  // pitch: of sums
  int passes, lanes, run;
  size_t rows, counts, parts;  // of 4 bytes
  EmbeddingPlan(int64_t n, int64_t V, int64_t D) {
    strips = (D + 511) / 512;
    // Rows of a piece: few, so that there are wavefronts enough, until the pieces' own starts and ends cost more (rows of 512 bf16, tokens as frequent as in a text, forward and gradient, 8, 16 and 32 rows:
    // of 8192 rows 36.5, 38.4 and 44.3 us, of 32768 65.2, 62.0 and 66.4, of 131072 159, 138 and 127).
    run = n * strips < 16384 ? 8 : (n * strips < 65536 ? 16 : 32);
    pieces = (n + run - 1) / run;
    for (lanes = 1; lanes < 64 && lanes * 8 < D;) lanes *= 2;
    passes = 0, blocks = 0;
    if (n > kCountedRows) {
      blocks = (n + kSortedRows - 1) / kSortedRows;
      for (int64_t v = V; v; v >>= kDigitBits) ++passes;  // (V itself stands for no token)
    }
    rows = (size_t)(n + 3) / 4 * 4;
    counts = (size_t)blocks * kDigits;
    pitch = (D + 7) / 8 * 8;
    parts = (size_t)pieces * (size_t)pitch;
  }
  size_t bytes() const { return (rows * (passes > 1 ? 4 : 2) + counts + 2 * parts) * 4; }
};

size_t rtn_embedding_bwd_workspace_bytes(int64_t rows, int64_t V, int64_t D, int32_t) {
  return rows <= 0 || V <= 0 || D <= 0 || rows > kMaxRows || V > kMaxRows ? 0 : EmbeddingPlan(rows, V, D).bytes();
}

int rtn_embedding_bwd(const int64_t* tokens, const void* dy, int64_t ld, void* Dtable, int64_t rows, int64_t V, int64_t D, int32_t dtype, float scale, void* workspace,
                      size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const char* what = "embedding gradient";
  const int rc = embedding_check(what, tokens, dy, &ld, Dtable, rows, V, D, dtype);
  if (rc != RTN_OK) return rc;
  if (!V || !D) return RTN_OK;
  if (!Dtable || (rows && (!tokens || !dy))) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  const EmbeddingPlan p(rows, V, D);
  const int e = size_of(dtype);
  if (D > INT64_MAX / 16 / V || D > INT64_MAX / 16 / (rows + 1) || D * V * e / kFilled >= max_blocks(1024) / 2 || p.strips > max_blocks(256) / 2 / (p.pieces + 1))
    return fail(RTN_ERR_SHAPE, "%s: %lld rows of a table [%lld,%lld] are too many for one call", what, (long long)rows, (long long)V, (long long)D);
  const int64_t bytes = D * V * e, filling = (bytes + kFilled - 1) / kFilled;
  const size_t need = rows ? p.bytes() : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  const hipStream_t stream = (hipStream_t)hip_stream;
  unsigned *now = (unsigned*)workspace, *other = now + 2 * p.rows, *counts = now + p.rows * (p.passes > 1 ? 4 : 2);
  EmbeddingArgs a{tokens, dy, ld, Dtable, rows, V, D, scale, nullptr, nullptr};
  if (p.passes) {
    SortArgs s{a, nullptr, nullptr, counts, (int)p.blocks, 0};
    // (each launch fills its share of the table)
    auto launch = [&](void (*kernel)(SortArgs, EmbeddingFill), int part) {
      const int64_t from = filling * part / (2 * p.passes), to = filling * (part + 1) / (2 * p.passes);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(p.blocks + to - from)), dim3(1024), 0, stream, s, EmbeddingFill{bytes, from});
    };
    for (int pass = 0; pass < p.passes; ++pass, s.shift += kDigitBits) {
      s.e.order = now, s.e.token_of = now + p.rows;
      launch(k_embedding_digits, 2 * pass);
      launch(k_embedding_move, 2 * pass + 1);
      s.order = s.e.order, s.token_of = s.e.token_of;
      std::swap(now, other);
    }
    a.order = s.e.order, a.token_of = s.e.token_of;
  } else {
    a.order = now, a.token_of = now + p.rows;
    const unsigned sorting = (unsigned)((rows + 15) / 16);
    hipLaunchKernelGGL(k_embedding_order, dim3(sorting + (unsigned)filling), dim3(1024), 0, stream, a, sorting, EmbeddingFill{bytes, 0});
  }
  const EmbeddingSumArgs s{a, (float*)(counts + p.counts), (float*)(counts + p.counts) + p.parts, p.pitch, (int)p.pieces, (int)p.strips, p.lanes, p.run};
  if (rows)
    with_type(dtype, [&](auto type) {
      typedef decltype(type) AT;
      hipLaunchKernelGGL(k_embedding_sums<AT>, dim3((unsigned)((p.pieces * p.strips * p.lanes + 255) / 256)), dim3(256), 0, stream, s);
      if (p.pieces > 1) hipLaunchKernelGGL(k_embedding_join<AT>, dim3((unsigned)((p.pieces * p.strips + 3) / 4)), dim3(256), 0, stream, s);
    });
  return launched(what);
}

// ---- beam search ----------------------------------------------------------------------------------------------------
// Pieces: all continuations of a search at once where they are few (64 searches of 8 hypotheses with 1000 scores, 8 of them: 7.9 us, in pieces 10.7).  Else pieces of hypotheses: short ones, several of
// which are on a compute unit at once, where one round joins their choices (256 searches of 12 with 32000 scores in bf16, 12 of them: 69 us, in long pieces 85); long ones, as long as a workgroup can hold,
// where there are too many of these (one search of 64 with 32000 scores, 64 of them: 20 us, in short pieces 29).
struct BeamPlan {
  int64_t splits, segment, lists;  // lists: of choices, per search, behind the first round
  BeamPlan(int32_t B, int32_t K, int64_t V, int32_t beam) {
    if (K * V <= kBeamFew) {
      splits = 1, segment = V, lists = 0;
      return;
    }
    splits = (V + kBeamLong - 1) / kBeamLong;
    if (const int64_t small = (V + kBeamShort - 1) / kBeamShort; K * small * beam <= kBeamJoined) splits = small;
    segment = ((V + splits - 1) / splits + 7) / 8 * 8;
    lists = K * splits;
  }
  size_t bytes(int32_t B, int32_t beam) const {  // two halves: a round reads one and writes the other
    const size_t first = (size_t)B * (size_t)lists * (size_t)beam * 8;
    return first + (lists > per(beam) ? (size_t)B * (size_t)((lists + per(beam) - 1) / per(beam)) * (size_t)beam * 8 : 0);
  }
  static int64_t per(int32_t beam) { return kBeamJoined / beam; }  // lists that are joined at once
};
static bool beam_valid(int32_t B, int32_t K, int64_t V, int32_t beam) { return B >= 0 && K >= 1 && V >= 1 && V <= kMaxScores && V <= INT32_MAX / K && beam >= 1 && beam <= kMaxBeam && beam <= K * V; }

size_t rtn_beam_select_workspace_bytes(int32_t B, int32_t K, int64_t V, int32_t, int32_t beam) { return beam_valid(B, K, V, beam) ? BeamPlan(B, K, V, beam).bytes(B, beam) : 0; }

int rtn_beam_select(const void* scores, int64_t ld, const float* totals, const uint8_t* ended, int64_t end_token, float* out_totals, int64_t* sources, int64_t* tokens,
                    int32_t B, int32_t K, int64_t V, int32_t dtype, int32_t beam, void* workspace, size_t workspace_bytes, void* hip_stream) {
  g_last_error.clear();
  const char* what = "beam selection";
  if (B < 0 || K < 1 || V < 1 || V > kMaxScores || V > INT32_MAX / K) return fail(RTN_ERR_SHAPE, "%s: %d searches of %d hypotheses with %lld scores", what, B, K, (long long)V);
  if (!known(dtype)) return fail(RTN_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  if (beam < 1 || beam > kMaxBeam || beam > K * V) return fail(RTN_ERR_RANGE, "%s: beam of %d from %d hypotheses with %lld scores (at most %d)", what, beam, K, (long long)V, kMaxBeam);
  if (ended && (end_token < 0 || end_token >= V)) return fail(RTN_ERR_RANGE, "%s: end token %lld of %lld", what, (long long)end_token, (long long)V);
  if (const int rc = pitch_check(what, "the scores", &ld, V); rc != RTN_OK) return rc;
  if (!B) return RTN_OK;
  if (!scores || !totals || !out_totals || !sources || !tokens) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  if (!aligned(scores, size_of(dtype)) || !aligned(totals, 4) || !aligned(out_totals, 4) || !aligned(sources, 8) || !aligned(tokens, 8))
    return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  const BeamPlan p(B, K, V, beam);
  const size_t need = p.bytes(B, beam);
  if (need && (!workspace || workspace_bytes < need)) return fail(RTN_ERR_WORKSPACE, "%s: workspace of %zu bytes needed", what, need);
  if (!aligned(workspace, 16)) return fail(RTN_ERR_ARG, "%s: workspace must be 16-byte aligned", what);
  if (std::max<int64_t>(p.lists, 1) > max_blocks(1024) / B) return fail(RTN_ERR_SHAPE, "%s: %d searches of %d hypotheses with %lld scores are too many for one call", what, B, K, (long long)V);
  BeamArgs a{scores, ld, totals, ended, end_token, out_totals, sources, tokens, B, K, beam, (int)V, (int)p.splits, (int)p.segment, (int)p.lists, 0, nullptr, (unsigned long long*)workspace};
  const hipStream_t stream = (hipStream_t)hip_stream;
  with_type(dtype, [&](auto type) {
    typedef decltype(type) AT;
    if (!p.lists) {
      if (K * V <= 2048)
        hipLaunchKernelGGL((k_beam_all<AT, 4, 8>), dim3((unsigned)B), dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((k_beam_all<AT, 16, 8>), dim3((unsigned)B), dim3(1024), 0, stream, a);
      return;
    }
    const dim3 grid((unsigned)(B * p.lists));
    if (p.segment <= kBeamShort)
      hipLaunchKernelGGL((k_beam_pieces<AT, 4, 32>), grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((k_beam_pieces<AT, 16, 32>), grid, dim3(1024), 0, stream, a);
    for (int64_t lists = p.lists;;) {
      const int64_t next = (lists + BeamPlan::per(beam) - 1) / BeamPlan::per(beam);
      a.lists = (int)lists, a.next = (int)next;
      unsigned long long* const other = (unsigned long long*)workspace + (a.to == workspace ? (size_t)B * (size_t)p.lists * (size_t)beam : 0);
      a.from = a.to, a.to = other;
      if (lists * beam <= 1024)
        hipLaunchKernelGGL((k_beam_join<4, 4>), dim3((unsigned)B), dim3(256), 0, stream, a);
      else
        hipLaunchKernelGGL((k_beam_join<16, kBeamJoined / 1024>), dim3((unsigned)(B * next)), dim3(1024), 0, stream, a);
      if (next == 1) break;
      lists = next;
    }
  });
  return launched(what);
}

int rtn_reorder_rows(int32_t count, const void* const* in, void* const* out, const int64_t* row_bytes, const int64_t* sources, int32_t B, int32_t K, int32_t beam,
                     void* hip_stream) {
  g_last_error.clear();
  const char* what = "reordering of rows";
  if (count < 0 || B < 0 || K < 0 || beam < 0) return fail(RTN_ERR_SHAPE, "%s: %d tensors of [%d,%d] to [%d,%d] rows", what, count, B, K, B, beam);
  if (!count || !B || !beam) return RTN_OK;
  if (!in || !out || !row_bytes || !sources) return fail(RTN_ERR_ARG, "%s: null pointer", what);
  if (!aligned(sources, 8)) return fail(RTN_ERR_ARG, "%s: misaligned pointer", what);
  const int64_t rows = (int64_t)B * beam;
  for (int n = 0; n < count; ++n) {
    if (row_bytes[n] < 0) return fail(RTN_ERR_SHAPE, "%s: rows of %lld bytes", what, (long long)row_bytes[n]);
    if (row_bytes[n] && ((K && !in[n]) || !out[n])) return fail(RTN_ERR_ARG, "%s: null pointer", what);
    if ((row_bytes[n] + kReorderPiece - 1) / kReorderPiece > max_blocks(256) / rows / kReordered)
      return fail(RTN_ERR_SHAPE, "%s: %lld rows of %lld bytes are too many for one call", what, (long long)rows, (long long)row_bytes[n]);
  }
  bool any = false;
  for (int first = 0; first < count; first += kReordered) {
    ReorderArgs a{{}, {}, {}, sources, B, K, beam, 1};
    const int some = std::min(count - first, kReordered);
    long long most = 0;
    for (int n = 0; n < some; ++n) {
      a.in[n] = (const char*)in[first + n], a.out[n] = (char*)out[first + n], a.bytes[n] = row_bytes[first + n];
      most = std::max(most, a.bytes[n]);
    }
    const int64_t pieces = (most + kReorderPiece - 1) / kReorderPiece;
    if (!pieces) continue;
    a.pieces = (int)pieces, any = true;
    hipLaunchKernelGGL(k_reorder_rows, dim3((unsigned)(rows * pieces), some), dim3(256), 0, (hipStream_t)hip_stream, a);
  }
  return any ? launched(what) : RTN_OK;
}

}  // extern "C"
