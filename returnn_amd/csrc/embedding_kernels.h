// gfx950 kernels of an embedding table: rows of tokens, scaled, and the table's gradient.
//
//   y_r = scale W[token_r],   dW[v] = scale sum_{r: token_r = v} dy_r, added in the order of r
#pragma once

#include "sequence_common.h"

namespace rtn {

struct EmbeddingArgs {
  const int64_t* tokens;
  const void* in;  // the table, or the errors
  long long ld;    // elements from one of its rows to the next
  void* out;
  long long rows;
  long long V;
  long long D;
  float scale;
  unsigned *order, *token_of;  // [rows]: rows in the order of their tokens, and these tokens
};

// Eight elements of a row per thread; those of a row's end one by one.
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding(EmbeddingArgs a) {
  const long long groups = (a.D + 7) / 8, item = blockIdx.x * 256ll + threadIdx.x;
  const long long r = item / groups, e = (item - r * groups) * 8;
  if (r >= a.rows) return;
  const long long token = a.tokens[r];
  const float none = token < 0 ? 0.f : __builtin_nanf("");
  const bool has = token >= 0 && token < a.V;
  const AT* from = (const AT*)a.in + (has ? token * a.ld : 0) + e;
  AT* to = (AT*)a.out + r * a.D + e;
  if (e + 8 <= a.D) {
    float v[8];
    Eight<AT> q;
    if (has) {
      q.load(from);
      q.get(v);
    }
    for (int k = 0; k < 8; ++k) v[k] = has ? v[k] * a.scale : none;
    q.set(v);
    q.store(to);
  } else {
    for (int k = 0; e + k < a.D; ++k) store_f32(to + k, has ? load_f32(from + k) * a.scale : none);
  }
}

// ---- the gradient: rows in the order of their tokens, then sums over runs of one token -------------------------------------

__device__ __forceinline__ unsigned token_key(const EmbeddingArgs& a, long long r) {
  const long long t = a.tokens[r];
  return t < 0 || t >= a.V ? (unsigned)a.V : (unsigned)t;  // (rows without a token come last)
}

// Where a row comes: after all of lower tokens and the earlier ones of the same, counted.  64 rows per workgroup, each of its 16 wavefronts counts among a 16th of all.
constexpr int kCountedRows = 8192;
__global__ __launch_bounds__(1024) void k_embedding_order(EmbeddingArgs a) {
  __shared__ alignas(16) unsigned keys[kCountedRows];
  __shared__ unsigned before_of[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = (int)a.rows, r = blockIdx.x * 64 + lane;
  const int padded = (rows + 63) / 64 * 64, part = padded / 16;  // (a multiple of 4)
  for (int i = threadIdx.x; i < padded; i += 1024) keys[i] = i < rows ? token_key(a, i) : 0xFFFFFFFFu;
  __syncthreads();
  const unsigned mine = r < rows ? keys[r] : 0;
  unsigned before = 0;
  for (int i = wave * part; i < (wave + 1) * part; i += 4) {
    const seq_u32x4 k = *(const seq_u32x4*)(keys + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) before += k[j] < mine + (i + j < r);
  }
  before_of[wave][lane] = before;
  __syncthreads();
  if (wave == 0 && r < rows) {
    before = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) before += before_of[w][lane];
    a.order[before] = (unsigned)r;
    a.token_of[before] = mine;
  }
}

// More rows: one pass for 8 bits of the token after the other, from the lowest on; each pass counts digits in blocks of rows, then every block moves its rows behind
// those of lower digits and those of earlier blocks.  Within a block a wavefront has 64 neighbouring rows at a time; lanes of one digit find each other by ballots.
constexpr int kDigits = 256, kSortedRows = 4096;  // rows of a block: 16 wavefronts with four times 64
struct SortArgs {
  EmbeddingArgs e;
  const unsigned *order, *token_of;  // of the pass before, or NULL: rows as they come
  unsigned* counts;                  // [blocks][digits]
  int blocks, shift;
};
__device__ __forceinline__ unsigned sort_key(const SortArgs& a, long long i) { return a.token_of ? a.token_of[i] : token_key(a.e, i); }
__global__ __launch_bounds__(1024) void k_embedding_digits(SortArgs a) {
  __shared__ unsigned count[kDigits];
  if (threadIdx.x < kDigits) count[threadIdx.x] = 0;
  __syncthreads();
  for (int n = 0; n < kSortedRows / 1024; ++n) {
    const long long i = (long long)blockIdx.x * kSortedRows + n * 1024 + threadIdx.x;
    if (i < a.e.rows) atomicAdd(&count[sort_key(a, i) >> a.shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kDigits) a.counts[(long long)blockIdx.x * kDigits + threadIdx.x] = count[threadIdx.x];
}
__global__ __launch_bounds__(1024) void k_embedding_move(SortArgs a) {
  __shared__ unsigned at_of[16][kDigits], all_of[4][kDigits], earlier_of[4][kDigits];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digit = threadIdx.x & (kDigits - 1), quarter = threadIdx.x / kDigits;
  unsigned all = 0, earlier = 0;
  for (int b = quarter; b < a.blocks; b += 4) {
    const unsigned n = a.counts[(long long)b * kDigits + digit];
    all += n, earlier += b < (int)blockIdx.x ? n : 0;
  }
  all_of[quarter][digit] = all, earlier_of[quarter][digit] = earlier;
  for (int w = threadIdx.x; w < 16 * kDigits; w += 1024) (&at_of[0][0])[w] = 0;
  __syncthreads();
  unsigned key[kSortedRows / 1024], row[kSortedRows / 1024], rank[kSortedRows / 1024];
#pragma unroll
  for (int n = 0; n < kSortedRows / 1024; ++n) {
    const long long i = (long long)blockIdx.x * kSortedRows + wave * (kSortedRows / 16) + n * 64 + lane;
    const bool in = i < a.e.rows;
    key[n] = in ? sort_key(a, i) : 0;
    row[n] = in ? (a.order ? a.order[i] : (unsigned)i) : 0xFFFFFFFFu;
    const unsigned d = key[n] >> a.shift & (kDigits - 1);
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const unsigned long long ones = __ballot(d >> bit & 1);
      same &= d >> bit & 1 ? ones : ~ones;
    }
    rank[n] = 0;
    if (in) {
      rank[n] = at_of[wave][d] + __popcll(same & ((1ull << lane) - 1));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (all have read before the first one adds)
      if ((same >> lane) == 1) at_of[wave][d] = rank[n] + 1;   // (the last one of a digit)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) {  // where the digits begin: four digits a lane
    unsigned of[4], sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      of[j] = sum;
      sum += all_of[0][lane * 4 + j] + all_of[1][lane * 4 + j] + all_of[2][lane * 4 + j] + all_of[3][lane * 4 + j];
    }
    unsigned up = sum;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const unsigned o = __shfl_up(up, step);
      if (lane >= step) up += o;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) all_of[0][lane * 4 + j] = up - sum + of[j];
  }
  __syncthreads();
  if (threadIdx.x < kDigits) {  // and the wavefronts' rows of them
    unsigned at = all_of[0][digit] + earlier_of[0][digit] + earlier_of[1][digit] + earlier_of[2][digit] + earlier_of[3][digit];
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const unsigned n = at_of[w][digit];
      at_of[w][digit] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kSortedRows / 1024; ++n)
    if (row[n] != 0xFFFFFFFFu) {
      const unsigned to = at_of[wave][key[n] >> a.shift & (kDigits - 1)] + rank[n];
      a.e.order[to] = row[n];
      a.e.token_of[to] = key[n];
    }
}

// Sums: a wavefront takes kRun rows in the order of their tokens and 512 columns.  A run of one token inside of them is a row of the table; of a run that goes on the sum so far is
// kept, of one that has begun before the sum of what is here.  The other wavefronts write the rows of the table that no token has.
constexpr int kRun = 32, kBare = 64;  // rows of a wavefront
struct EmbeddingSumArgs {
  EmbeddingArgs e;
  float *begun, *rest;  // [pieces][D]
  int pieces, strips;
  long long sums;  // wavefronts of them
};
template <typename AT>
__device__ __forceinline__ void embedding_put(AT* to, int left, const float (&v)[8], float scale) {
  if (left >= 8) {
    float w[8];
    for (int k = 0; k < 8; ++k) w[k] = v[k] * scale;
    Eight<AT> q;
    q.set(w);
    q.store_streamed(to);
  } else {
    for (int k = 0; k < 8; ++k)
      if (k < left) store_f32(to + k, v[k] * scale);
  }
}
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding_sums(EmbeddingSumArgs s) {
  const EmbeddingArgs& a = s.e;
  const int lane = threadIdx.x & 63;
  const long long item = blockIdx.x * 4ll + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned V = (unsigned)a.V;
  if (item >= s.sums) {
    const long long v0 = (item - s.sums) * kBare, v = v0 + lane;
    if (v0 >= a.V) return;
    unsigned lo = 0, hi = (unsigned)a.rows;
    while (lo < hi) {  // (as many turns in all lanes, or one fewer)
      const unsigned mid = lo + (hi - lo) / 2;
      if (a.token_of[mid] < (unsigned)v)
        lo = mid + 1;
      else
        hi = mid;
    }
    unsigned long long bare = __ballot(v < a.V && !(lo < a.rows && a.token_of[lo] == (unsigned)v));
    const float none[8] = {};
    for (; bare; bare &= bare - 1) {
      AT* to = (AT*)a.out + (v0 + __builtin_ctzll(bare)) * a.D;
      for (long long e = lane * 8; e < a.D; e += 512) embedding_put(to + e, (int)(a.D - e < 8 ? a.D - e : 8), none, 0.f);
    }
    return;
  }
  const int piece = (int)(item / s.strips), strip = (int)(item - (long long)piece * s.strips);
  const long long col = strip * 512ll + lane * 8, first = (long long)piece * kRun;
  const int left = (int)(a.D - col < 0 ? 0 : (a.D - col < 8 ? a.D - col : 8)), rows = (int)(a.rows - first < kRun ? a.rows - first : kRun);
  const unsigned before = first ? a.token_of[first - 1] : 0xFFFFFFFFu, after = first + rows < a.rows ? a.token_of[first + rows] : 0xFFFFFFFFu;
  float sum[8] = {};
  unsigned token = a.token_of[first];
  bool begun_here = token != before;
  auto flush = [&](bool ends_here) {
    if (token >= V || left == 0) return;
    if (begun_here && ends_here) {
      embedding_put((AT*)a.out + token * a.D + col, left, sum, a.scale);
    } else {
      // (a run that fills this piece and goes on is part of the run that began earlier)
      float* to = (begun_here ? s.begun : s.rest) + piece * a.D + col;
      for (int k = 0; k < 8; ++k)
        if (k < left) to[k] = sum[k];
    }
  };
  constexpr int AHEAD = 8;
  for (int p0 = 0; p0 < rows; p0 += AHEAD) {
    Eight<AT> q[AHEAD];
    unsigned key[AHEAD];
    float part[AHEAD][8];
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      const long long at = first + (p0 + p < rows ? p0 + p : rows - 1);
      key[p] = a.token_of[at];
      const AT* from = (const AT*)a.in + a.order[at] * a.ld + col;
      const bool wanted = p0 + p < rows && key[p] < V;
      if (wanted && left == 8) {
        q[p].load(from);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) part[p][k] = wanted && k < left ? load_f32(from + k) : 0.f;
        q[p].set(part[p]);
      }
    }
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      if (p0 + p >= rows) break;
      if (key[p] != token) {
        flush(true);
        token = key[p], begun_here = true;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = 0.f;
      }
      q[p].get(part[p]);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += part[p][k];
    }
  }
  flush(token != after);
}

// Rows of the table whose run goes over several pieces.
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding_join(EmbeddingSumArgs s) {
  const EmbeddingArgs& a = s.e;
  const int lane = threadIdx.x & 63;
  const long long item = blockIdx.x * 4ll + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= s.sums) return;
  const int piece = (int)(item / s.strips), strip = (int)(item - (long long)piece * s.strips);
  const long long col = strip * 512ll + lane * 8, first = (long long)piece * kRun, next = first + kRun;
  if (next >= a.rows) return;
  const unsigned token = a.token_of[next];
  // (the run has to go on behind this piece, and to begin in it)
  if (token >= (unsigned)a.V || a.token_of[next - 1] != token || (first && a.token_of[first - 1] == token)) return;
  long long lo = next, hi = a.rows;
  while (lo < hi) {
    const long long mid = lo + (hi - lo) / 2;
    if (a.token_of[mid] == token)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int last = (int)((lo - 1) / kRun), left = (int)(a.D - col < 0 ? 0 : (a.D - col < 8 ? a.D - col : 8));
  if (left == 0) return;
  float sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) sum[k] = k < left ? s.begun[piece * a.D + col + k] : 0.f;
#pragma unroll 4
  for (int p = piece + 1; p <= last; ++p)
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += k < left ? s.rest[p * a.D + col + k] : 0.f;
  embedding_put((AT*)a.out + token * a.D + col, left, sum, a.scale);
}

}  // namespace rtn
