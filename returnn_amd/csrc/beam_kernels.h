// gfx950 kernels of a step of beam search: the best continuations of all hypotheses of a search, and the rows of states that go with them.
//
//   joint[b,k,v] = totals[b,k] + scores[b,k,v], one addition in float32; the scores of a hypothesis that has ended are 0 for the end token and -inf for all others
#pragma once

#include "token_order.h"

namespace rtn {

constexpr int kMaxBeam = 64;
constexpr long long kMaxScores = 1 << 26;  // of a hypothesis: pieces are a multiple of 8 long, and where the last one begins is a 32-bit number
constexpr int kBeamFew = 8192;                      // continuations of a search that one workgroup takes at once
constexpr int kBeamShort = 8192, kBeamLong = 32768;  // of a piece
constexpr int kBeamJoined = 4096;                   // choices that are joined at once

struct BeamArgs {
  const void* scores;
  long long ld;
  const float* totals;
  const unsigned char* ended;
  long long end_token;
  float* out_totals;
  int64_t *sources, *tokens;
  int B, K, beam, V;
  int splits, segment;  // pieces of a hypothesis' scores, and how long they are
  int lists, next;      // of choices, per search, that there are and that are to be
  const unsigned long long* from;
  unsigned long long* to;  // [B][lists][beam], each in descending order, 0 where there are no more
};

__device__ __forceinline__ void put_choice(const BeamArgs& a, int b, int rank, unsigned long long q) {
  const unsigned index = ~(unsigned)q, source = index / (unsigned)a.V;
  const long long at = (long long)b * a.beam + rank;
  a.out_totals[at] = logit_of(q);
  a.sources[at] = source;
  a.tokens[at] = index - source * (unsigned)a.V;
}

// The best `beam` of what a workgroup of W wavefronts holds, E per thread: high[e] the place in the order of sums (0: nothing), low(e) the lower half of the number that
// orders them all, in which no two are alike; ordered(e): whether low falls from thread to thread and from e to e, eight at a time, so that equal sums are met lowest index first.
// put(rank, number) for the ranks below `beam`; how many there were.
//
// All are read once and stay in registers.  A bound from below is the beam-th largest of 64 or 256 groups' largest; what reaches it is listed and finds its rank.  Where that is too much, it is mostly equal to the bound
// (hypotheses that are none, all at minus infinity): then what is above it is listed, and the first ones that are equal follow.  Else the beam-th largest is found digit by digit.
constexpr int kBeamListed = 512;
template <int W>
struct BeamScratch {
  unsigned long long list[kBeamListed];
  alignas(16) unsigned groups[W < 16 ? 256 : 1024];
  unsigned digits[256];
  unsigned bound, listed, waves[W];
  unsigned long long prefix;
  int wanted;
};
template <int W, int E, typename Low, typename Put>
__device__ __forceinline__ int beam_best(BeamScratch<W>& s, const unsigned (&high)[E], Low low, int beam, bool in_order, Put put) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, thread = threadIdx.x;
  unsigned most = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) most = high[e] > most ? high[e] : most;
  s.groups[thread] = most;
  if (thread == 0) s.listed = 0, s.bound = 0xFFFFFFFFu;
  __syncthreads();
  const int groups = beam <= 32 ? 64 : 256;
  if (thread < groups) {
    unsigned mine = 0;
    for (int o = thread; o < 64 * W; o += groups) mine = s.groups[o] > mine ? s.groups[o] : mine;
    most = mine;
  }
  __syncthreads();
  if (thread < groups) s.groups[thread] = most;
  __syncthreads();
  if (thread < groups) {
    int larger = 0;
#pragma unroll 4
    for (int o = 0; o < groups; o += 4) {
      const seq_u32x4 four = *(const seq_u32x4*)(s.groups + o);
#pragma unroll
      for (int j = 0; j < 4; ++j) larger += four[j] > most;
    }
    const unsigned least = wave_min(larger < beam ? most : 0xFFFFFFFFu);
    if (lane == 0) atomicMin(&s.bound, least);
  }
  __syncthreads();
  unsigned bound = s.bound;
  if (bound == 0) bound = 1;  // (not what is nothing)
  auto make_list = [&](unsigned least) {
    unsigned hits = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) hits += high[e] >= least;
    if (hits) {
      unsigned at = atomicAdd(&s.listed, hits);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (high[e] >= least) {
          if (at < kBeamListed) s.list[at] = (unsigned long long)high[e] << 32 | low(e);
          ++at;
        }
    }
    __syncthreads();
    return (int)s.listed;
  };
  // (16 lanes for each of the list)
  auto rank_list = [&](int n) {
    for (int j = thread >> 4; j < n; j += 4 * W) {
      const unsigned long long mine = s.list[j];
      const int rank = rank_in(s.list, n, mine, lane);
      if ((lane & 15) == 0 && rank < beam) put(rank, mine);
    }
  };
  int n = make_list(bound);
  if (n <= kBeamListed) {
    rank_list(n);
    return n < beam ? n : beam;
  }
  __syncthreads();
  if (thread == 0) s.listed = 0;
  __syncthreads();
  n = bound == 0xFFFFFFFFu ? 0 : make_list(bound + 1);
  if (n < beam && in_order) {
    rank_list(n);
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      unsigned hits = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) hits += high[8 * j + k] == bound;
      unsigned up = hits;
#pragma unroll
      for (int step = 1; step < 64; step *= 2) {
        const unsigned o = __shfl_up(up, step);
        if (lane >= step) up += o;
      }
      if (lane == 63) s.waves[wave] = up;
      __syncthreads();
      int rank = n + (int)(up - hits);
      for (int w = 0; w < W; ++w) rank += w < wave ? s.waves[w] : 0, n += s.waves[w];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (high[8 * j + k] == bound) {
          if (rank < beam) put(rank, (unsigned long long)bound << 32 | low(8 * j + k));
          ++rank;
        }
      if (n >= beam) return beam;
      __syncthreads();
    }
    return n;
  }
  if (thread == 0) s.prefix = 0, s.wanted = beam;
  for (int shift = 56; shift >= 0; shift -= 8) {
    __syncthreads();
    if (thread < 256) s.digits[thread] = 0;
    __syncthreads();
    const unsigned long long prefix = s.prefix;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const unsigned long long q = (unsigned long long)high[e] << 32 | low(e);
      if (shift == 56 || q >> (shift + 8) == prefix) atomicAdd(&s.digits[q >> shift & 255], 1u);
    }
    __syncthreads();
    if (thread == 0) {
      int digit = 255, wanted = s.wanted;
      while (digit && (int)s.digits[digit] < wanted) wanted -= s.digits[digit--];
      s.prefix = prefix << 8 | (unsigned)digit, s.wanted = wanted;
    }
  }
  __syncthreads();
  const unsigned long long least = s.prefix;
  if (thread == 0) s.listed = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const unsigned long long q = (unsigned long long)high[e] << 32 | low(e);
    if (q >= least) s.list[atomicAdd(&s.listed, 1u)] = q;  // (`beam` of them: no two are alike)
  }
  __syncthreads();
  rank_list(beam);
  return beam;
}

// All continuations of a search, one workgroup each: number (e / 8 * 64 W + thread) * 8 + e % 8 of them.
template <typename AT, int W, int E>
__global__ __launch_bounds__(64 * W) void k_beam_all(BeamArgs a) {
  __shared__ BeamScratch<W> scratch;
  const int b = blockIdx.x, all = a.K * a.V;
  unsigned high[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = (e / 8 * 64 * W + (int)threadIdx.x) * 8 + e % 8;
    high[e] = 0;
    if (at < all) {
      const int k = (unsigned)at / (unsigned)a.V, v = at - k * a.V;
      const long long row = (long long)b * a.K + k;
      const float s = a.ended && a.ended[row] ? (v == a.end_token ? 0.f : -__builtin_inff()) : load_f32((const AT*)a.scores + row * a.ld + v);
      high[e] = order_of(a.totals[row] + s);
    }
  }
  beam_best<W, E>(
      scratch, high, [&](int e) { return ~(unsigned)((e / 8 * 64 * W + (int)threadIdx.x) * 8 + e % 8); }, a.beam, true, [&](int rank, unsigned long long q) { put_choice(a, b, rank, q); });
}

// A piece of a hypothesis' continuations per workgroup.  Bound by memory where there are many (108 MB in 25-27 us, 4.2 TB/s: workgroups have no load in flight while they list and rank, but several are on a compute unit), else by
// the latency of one load, a few rounds of LDS and barriers (6.2-6.7 us).
template <typename AT, int W, int E>
__global__ __launch_bounds__(64 * W) void k_beam_pieces(BeamArgs a) {
  __shared__ BeamScratch<W> scratch;
  const long long row = blockIdx.x / (unsigned)a.splits;
  const int split = (int)(blockIdx.x - (unsigned)row * a.splits), k = (int)((unsigned)row % (unsigned)a.K);
  const int v0 = split * a.segment, v1 = v0 + a.segment < a.V ? v0 + a.segment : a.V;
  const float total = a.totals[row];
  const bool ended = a.ended && a.ended[row];
  const AT* scores = (const AT*)a.scores + row * a.ld;
  unsigned long long* to = a.to + (long long)blockIdx.x * a.beam;
  if (ended && total < __builtin_inff()) {  // (nothing to look for: the end, unless that is at minus infinity as well, and the lowest tokens)
    const int end = (int)a.end_token, first = end >= v0 && end < v1 && total > -__builtin_inff();
    if ((int)threadIdx.x < a.beam) {
      int v = v0 + (int)threadIdx.x - first;
      if (first && v >= end) ++v;
      to[threadIdx.x] = first && threadIdx.x == 0 ? alternative(total, (unsigned)(k * a.V + end)) : (v < v1 ? alternative(-__builtin_inff(), (unsigned)(k * a.V + v)) : 0);
    }
    return;
  }
  unsigned high[E];
  auto own = [&](int j) { return v0 + (j * 64 * W + (int)threadIdx.x) * 8; };
  if (!ended) {
    Eight<AT> q[E / 8];
#pragma unroll
    for (int j = 0; j < E / 8; ++j)
      if (own(j) + 8 <= v1) q[j].load(scores + own(j));
#pragma unroll
    for (int j = 0; j < E / 8; ++j) {
      float v[8];
      if (own(j) + 8 <= v1) {
        q[j].get(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) high[8 * j + i] = order_of(total + v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) high[8 * j + i] = own(j) + i < v1 ? order_of(total + load_f32(scores + own(j) + i)) : 0;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int v = own(e / 8) + e % 8;
      high[e] = v < v1 ? order_of(total + (v == a.end_token ? 0.f : -__builtin_inff())) : 0;
    }
  }
  const int n = beam_best<W, E>(
      scratch, high, [&](int e) { return ~(unsigned)(k * a.V + own(e / 8) + e % 8); }, a.beam, true, [&](int rank, unsigned long long q) { to[rank] = q; });
  for (int rank = n + threadIdx.x; rank < a.beam; rank += 64 * W) to[rank] = 0;
}

// Choices of several lists joined: to one list, or to the search's.
template <int W, int E>
__global__ __launch_bounds__(64 * W) void k_beam_join(BeamArgs a) {
  __shared__ BeamScratch<W> scratch;
  const int b = blockIdx.x / (unsigned)a.next, part = (int)(blockIdx.x - (unsigned)b * a.next), per = kBeamJoined / a.beam;
  const int lists = a.lists - part * per < per ? a.lists - part * per : per;
  const unsigned long long* from = a.from + ((long long)b * a.lists + part * per) * a.beam;
  // The first of all lists, then the second of all: so the groups of beam_best have their shares of the best.  (List by list the first ones of 64 lists of 64 were in 4 of the 256 groups, their bound
  // let hundreds through, and the choice was made digit by digit: one search of 64 hypotheses with 32000 scores, 64 of them: 77 us, so 29.)
  unsigned high[E], low[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int at = e * 64 * W + threadIdx.x, rank = (unsigned)at / (unsigned)lists, list = at - rank * lists;
    const unsigned long long q = rank < a.beam ? from[list * a.beam + rank] : 0;
    high[e] = (unsigned)(q >> 32), low[e] = (unsigned)q;
  }
  unsigned long long* to = a.to + ((long long)b * a.next + part) * a.beam;
  const int n = beam_best<W, E>(
      scratch, high, [&](int e) { return low[e]; }, a.beam, false, [&](int rank, unsigned long long q) {
        if (a.next > 1)
          to[rank] = q;
        else
          put_choice(a, b, rank, q);
      });
  if (a.next > 1)
    for (int rank = n + threadIdx.x; rank < a.beam; rank += 64 * W) to[rank] = 0;
}

constexpr int kReordered = 16;        // tensors of one launch
constexpr int kReorderPiece = 16384;  // bytes of a row that a workgroup moves
struct ReorderArgs {
  const char* in[kReordered];
  char* out[kReordered];
  long long bytes[kReordered];  // of a row
  const int64_t* sources;
  int B, K, beam;
  int pieces;
};

// Part of a row per workgroup, several tensors in a launch; bound by memory (203 MB in 35 us, 5.8 TB/s; some of it is still in the Infinity Cache) or a launch (3 us): 16 bytes a thread where addresses and rows allow it, else 4, else 1.
template <typename T>
__device__ __forceinline__ void reorder_piece(const char* from, char* to, long long bytes, bool has) {
  constexpr int EACH = kReorderPiece / 256 / (int)sizeof(T) < 4 ? kReorderPiece / 256 / (int)sizeof(T) : 4;
  const int n = (int)(bytes / (int)sizeof(T));
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * EACH) {
    T v[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = has && i0 + j * 256 < n ? ((const T*)from)[i0 + j * 256] : T{};
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (i0 + j * 256 < n) __builtin_nontemporal_store(v[j], (T*)to + i0 + j * 256);
  }
}
__global__ __launch_bounds__(256) void k_reorder_rows(ReorderArgs a) {
  const int row = blockIdx.x / (unsigned)a.pieces, piece = blockIdx.x - row * a.pieces, n = blockIdx.y, b = row / a.beam;
  const long long whole = a.bytes[n], start = (long long)piece * kReorderPiece;
  if (start >= whole) return;
  const int64_t source = a.sources[row];
  const bool has = source >= 0 && source < a.K;
  const long long bytes = whole - start < kReorderPiece ? whole - start : kReorderPiece;
  const char* from = a.in[n] + ((long long)b * a.K + (has ? source : 0)) * whole + start;
  char* to = a.out[n] + row * whole + start;
  const unsigned long long all = (unsigned long long)a.in[n] | (unsigned long long)a.out[n] | (unsigned long long)whole;
  if (all % 16 == 0)
    reorder_piece<seq_u32x4>(from, to, bytes, has);
  else if (all % 4 == 0)
    reorder_piece<unsigned>(from, to, bytes, has);
  else
    reorder_piece<unsigned char>(from, to, bytes, has);
}

}  // namespace rtn
