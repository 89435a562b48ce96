// gfx950 kernels of a step of beam search: the best continuations of all hypotheses of a search, and the rows of states that go with them.
//
//   joint[b,k,v] = totals[b,k] + scores[b,k,v], one addition in float32; of a hypothesis that has ended totals[b,k] for the end token and -inf for all others
#pragma once

#include "token_order.h"

namespace rtn {

constexpr int kMaxBeam = 64;

struct BeamArgs {
  const void* scores;
  long long ld;
  const float* totals;
  const unsigned char* ended;
  long long end_token;
  float* out_totals;
  int64_t *sources, *tokens;
  int B, K, beam;
  long long V;
  int splits;   // pieces of a hypothesis' scores
  long long segment;  // scores of a piece
  unsigned long long* part;  // [B][K][splits][beam]
};

__device__ __forceinline__ void put_choice(const BeamArgs& a, int b, int rank, unsigned long long q) {
  const unsigned index = ~(unsigned)q, source = (unsigned)(index / a.V);
  const long long at = (long long)b * a.beam + rank;
  a.out_totals[at] = logit_of(q);
  a.sources[at] = source;
  a.tokens[at] = index - source * a.V;
}

// One search per workgroup, one choice after the other.
template <typename AT>
__global__ __launch_bounds__(256) void k_beam_select(BeamArgs a) {
  __shared__ unsigned long long best_of[4];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  unsigned long long last = ~0ull;
  for (int rank = 0; rank < a.beam; ++rank) {
    unsigned long long best = 0;
    for (int k = 0; k < a.K; ++k) {
      const long long row = (long long)b * a.K + k;
      const float total = a.totals[row];
      const bool ended = a.ended && a.ended[row];
      for (long long v = threadIdx.x; v < a.V; v += 256) {
        const float s = ended ? (v == a.end_token ? 0.f : -__builtin_inff()) : load_f32((const AT*)a.scores + row * a.ld + v);
        const unsigned long long q = alternative(total + s, (unsigned)(k * a.V + v));
        best = q < last && q > best ? q : best;
      }
    }
    best = wave_max(best);
    if (lane == 0) best_of[wave] = best;
    __syncthreads();
    last = 0;
    for (int w = 0; w < 4; ++w) last = best_of[w] > last ? best_of[w] : last;
    if (threadIdx.x == 0) put_choice(a, b, rank, last);
    __syncthreads();
  }
}

constexpr int kReordered = 16;  // tensors of one launch
struct ReorderArgs {
  const char* in[kReordered];
  char* out[kReordered];
  long long bytes[kReordered];  // of a row
  const int64_t* sources;
  int B, K, beam;
  int count;
};

// One row per workgroup and tensor, byte by byte where it is not in words.
__global__ __launch_bounds__(256) void k_reorder_rows(ReorderArgs a) {
  const int row = blockIdx.x, n = blockIdx.y, b = row / a.beam;
  const int64_t source = a.sources[row];
  const bool has = source >= 0 && source < a.K;
  const long long bytes = a.bytes[n];
  const char* from = a.in[n] + ((long long)b * a.K + (has ? source : 0)) * bytes;
  char* to = a.out[n] + row * bytes;
  for (long long i = threadIdx.x; i < bytes; i += 256) to[i] = has ? from[i] : 0;
}

}  // namespace rtn
