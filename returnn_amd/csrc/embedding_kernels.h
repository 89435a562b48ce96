// gfx950 kernels of an embedding table: rows of tokens, scaled, and the table's gradient.
//
//   y_r = scale W[token_r],   dW[v] = scale sum_{r: token_r = v} dy_r, added in the order of r by blocks of them
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

// Eight elements of a row per thread; those of a row's end one by one.  Bound by memory: the largest measured call moves 99 MB in 18-20 us, 5.2 TB/s; few rows by a launch (2.2 us).
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

// Zeros for all of the table, by the workgroups behind the `first` of a launch, while these sort: rows that tokens have are written again, at most as many as there are tokens.
constexpr long long kFilled = 1 << 16;  // bytes for each of them
struct EmbeddingFill {
  long long bytes, from;  // of the table, and how many workgroups of earlier launches have been at it
};
__device__ __forceinline__ void embedding_fill(const EmbeddingArgs& a, unsigned first, EmbeddingFill fill) {
  const long long bytes = fill.bytes;
  char* to = (char*)a.out;
  // (whole words of 16 bytes; what is before and behind them, byte by byte)
  const long long head = ((16 - (long long)((unsigned long long)to & 15)) & 15) < bytes ? (16 - (long long)((unsigned long long)to & 15)) & 15 : bytes, words = (bytes - head) / 16;
  const long long start = (fill.from + (blockIdx.x - first)) * (kFilled / 16);
  const seq_u32x4 none = {0, 0, 0, 0};
  for (int i = threadIdx.x; i < kFilled / 16; i += 1024)
    if (start + i < words) __builtin_nontemporal_store(none, (seq_u32x4*)(to + head) + start + i);
  if (start == 0 && threadIdx.x < 32) {
    const long long tail = head + words * 16 + threadIdx.x - 16;
    if (threadIdx.x < 16 ? (long long)threadIdx.x < head : tail < bytes) to[threadIdx.x < 16 ? (long long)threadIdx.x : tail] = 0;
  }
}

// Where a row comes: after all of lower tokens and the earlier ones of the same, counted.  16 rows per workgroup, each against a 64th of all by 64 threads.  One launch in place of four for two digits:
// 1000, 4096 and 8192 rows of 512 bf16, forward and gradient, 20, 25 and 37 us, with digits 29, 37 and 43.  Bound by its comparisons, beside which the table's zeros are written.
constexpr int kCountedRows = 8192;
__global__ __launch_bounds__(1024) void k_embedding_order(EmbeddingArgs a, unsigned sorting, EmbeddingFill fill) {
  __shared__ alignas(16) unsigned keys[kCountedRows];
  __shared__ unsigned before_of[16][16];
  if (blockIdx.x >= sorting) return embedding_fill(a, sorting, fill);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = (int)a.rows, r = blockIdx.x * 16 + (lane & 15);
  const int padded = (rows + 255) / 256 * 256, part = padded / 64, first = (int)(threadIdx.x >> 4) * part;  // (a multiple of 4)
  for (int i = threadIdx.x; i < padded; i += 1024) keys[i] = i < rows ? token_key(a, i) : 0xFFFFFFFFu;
  __syncthreads();
  const unsigned mine = r < rows ? keys[r] : 0;
  unsigned before = 0;
  if (first + part <= (int)blockIdx.x * 16 || first >= (int)blockIdx.x * 16 + 16) {  // (all of the part on one side of the workgroup's rows)
    const unsigned below = mine + (first < (int)blockIdx.x * 16);
    for (int i = first; i < first + part; i += 4) {
      const seq_u32x4 k = *(const seq_u32x4*)(keys + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) before += k[j] < below;
    }
  } else {
    for (int i = first; i < first + part; ++i) before += keys[i] < mine + (i < r);
  }
  before += __shfl_xor(before, 16);
  before += __shfl_xor(before, 32);
  if (lane < 16) before_of[wave][lane] = before;
  __syncthreads();
  if (threadIdx.x < 16 && r < rows) {
    before = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) before += before_of[w][lane];
    a.order[before] = (unsigned)r;
    a.token_of[before] = mine;
  }
}

// More rows: one pass for 9 bits of the token after the other, from the lowest on; each pass counts digits in blocks of rows, then every block moves its rows behind
// those of lower digits and those of earlier blocks.  Within a block a wavefront has 64 neighbouring rows at a time; lanes of one digit find each other by ballots.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kSortedRows = 4096;  // rows of a block: 16 wavefronts with four times 64
struct SortArgs {
  EmbeddingArgs e;
  const unsigned *order, *token_of;  // of the pass before, or NULL: rows as they come
  unsigned* counts;                  // [blocks][digits]
  int blocks, shift;
};
__device__ __forceinline__ unsigned sort_key(const SortArgs& a, long long i) { return a.token_of ? a.token_of[i] : token_key(a.e, i); }
__global__ __launch_bounds__(1024) void k_embedding_digits(SortArgs a, EmbeddingFill fill) {
  __shared__ unsigned count[kDigits];
  if (blockIdx.x >= (unsigned)a.blocks) return embedding_fill(a.e, a.blocks, fill);
  if (threadIdx.x < kDigits) count[threadIdx.x] = 0;
  __syncthreads();
  for (int n = 0; n < kSortedRows / 1024; ++n) {
    const long long i = (long long)blockIdx.x * kSortedRows + n * 1024 + threadIdx.x;
    if (i < a.e.rows) atomicAdd(&count[sort_key(a, i) >> a.shift & (kDigits - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < kDigits) a.counts[(long long)blockIdx.x * kDigits + threadIdx.x] = count[threadIdx.x];
}
__global__ __launch_bounds__(1024) void k_embedding_move(SortArgs a, EmbeddingFill fill) {
  __shared__ unsigned at_of[16][kDigits], all_of[2][kDigits], earlier_of[2][kDigits];
  if (blockIdx.x >= (unsigned)a.blocks) return embedding_fill(a.e, a.blocks, fill);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, digit = threadIdx.x & (kDigits - 1), half = threadIdx.x / kDigits;
  unsigned all = 0, earlier = 0;
  for (int b = half; b < a.blocks; b += 2) {
    const unsigned n = a.counts[(long long)b * kDigits + digit];
    all += n, earlier += b < (int)blockIdx.x ? n : 0;
  }
  all_of[half][digit] = all, earlier_of[half][digit] = earlier;
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
    for (int bit = 0; bit < kDigitBits; ++bit) {
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
  if (threadIdx.x < 64) {  // where the digits begin: eight digits a lane
    unsigned of[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      of[j] = sum;
      sum += all_of[0][lane * 8 + j] + all_of[1][lane * 8 + j];
    }
    unsigned up = sum;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const unsigned o = __shfl_up(up, step);
      if (lane >= step) up += o;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) all_of[0][lane * 8 + j] = up - sum + of[j];
  }
  __syncthreads();
  if (threadIdx.x < kDigits) {  // and the wavefronts' rows of them
    unsigned at = all_of[0][digit] + earlier_of[0][digit] + earlier_of[1][digit];
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

// Sums: the rows of a token, in order, are cut into blocks of `run` from the token's first row on, so that how they are added does not depend on the rows of other tokens.  Up to 64 lanes, of 8 columns
// each, take the blocks that begin in `run` places of the sorted rows: one that goes on from an earlier place at most, then tokens' first ones, of which the last may have more behind it.  The sum of all rows of a token
// is a row of the table; those of a block with others before or behind it are kept, and joined in order.
// Eight rows are on their way at a time, and no atomics are needed, whose order would change sums.  Bound by memory: the largest measured call moves 73 MB in 19-20 us; few rows by latency (6 us,
// 9-10 where runs go over several pieces: where they begin is looked for first).
struct EmbeddingSumArgs {
  EmbeddingArgs e;
  float *begun, *rest;  // [pieces][pitch]
  long long pitch;      // D and what it lacks to a multiple of 8
  int pieces, strips;
  int lanes;  // of a piece and strip: a power of two
  int run;
};
template <typename AT>
__device__ __forceinline__ void embedding_put(AT* to, int left, const float (&v)[8], float scale) {
  if (left >= 8) {
    float w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = v[k] * scale;
    Eight<AT> q;
    q.set(w);
    q.store_streamed(to);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) store_f32(to + k, v[k] * scale);
  }
}
// Where the run of the token at `first - 1` begins, which is the token at `first` too.  A wavefront looks at 64 places at a time: the nearest ones and every 65th behind them at once, then ever wider apart
// while all are the token's, then between two of them.  (Of a run of up to 64 rows one round of loads, of up to 4224 two, of up to 278848 four.)
__device__ __forceinline__ long long embedding_run_begin(const EmbeddingArgs& a, long long first, unsigned token) {
  const int lane = threadIdx.x & 63;
  // (how many of the places at - step, at - 2 step, .. are the token's, of 64 that are above `above`)
  auto place_of = [&](long long at, long long step) { return at - step * (lane + 1); };
  auto key_of = [&](long long place, long long above) { return a.token_of[place > above ? place : first]; };
  auto count = [&](long long place, long long above, unsigned key) {
    const unsigned long long other = ~__ballot(place > above && key == token);
    return other ? __builtin_ctzll(other) : 64;
  };
  long long in = first - 1, out = -1, step = 65;  // the lowest place known to be the token's, and the highest known not to be
  const long long near = place_of(in, 1), far = place_of(in - 64, step);
  const unsigned near_key = key_of(near, -1), far_key = key_of(far, -1);
  int n = count(near, -1, near_key);
  if (n < 64) return in - n;
  in -= 64;
  auto look = [&]() { return count(place_of(in, step), out, key_of(place_of(in, step), out)); };
  for (n = count(far, -1, far_key);; n = look()) {
    in -= step * n;
    if (n < 64) break;
    step *= 65;
  }
  out = in - step < -1 ? -1 : in - step;
  while (in - out > 1) {
    step = (in - out - 1) / 65 + 1;
    n = look();
    in -= step * n;
    if (n < 64 && in - step > out) out = in - step;
  }
  return in;
}
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding_sums(EmbeddingSumArgs s) {
  const EmbeddingArgs& a = s.e;
  const long long item = (blockIdx.x * 256ll + threadIdx.x) / s.lanes;
  const int piece = (int)(item / s.strips), strip = (int)(item - (long long)piece * s.strips);
  const unsigned V = (unsigned)a.V, kEnd = 0xFFFFFFFFu;  // (no token)
  const long long col = ((long long)strip * s.lanes + threadIdx.x % s.lanes) * 8, first = (long long)piece * s.run, end = first + s.run;
  const int left = (int)(a.D - col < 0 ? 0 : (a.D - col < 8 ? a.D - col : 8));
  auto key_at = [&](long long place) {
    const unsigned key = a.token_of[place < a.rows ? place : a.rows - 1];
    return place < a.rows ? key : kEnd;
  };
  unsigned token = key_at(first);
  const unsigned before = first ? key_at(first - 1) : kEnd;
  long long place = first, begin = first;  // of the row, and of its block
  bool whole = true;                       // whether the block is its token's first one
  // (a wavefront's pieces, if it has several, are neighbours: one search for all that begin inside of the same run)
  const bool inside = token < V && before == token;
  long long run_begin = first;
  for (unsigned long long wanted = __ballot(inside); wanted;) {
    const int lane = __builtin_ctzll(wanted);
    const unsigned of = (unsigned)__builtin_amdgcn_readlane((int)token, lane);
    const long long found = embedding_run_begin(a, (long long)__builtin_amdgcn_readlane(piece, lane) * s.run, of);
    const bool mine = inside && token == of;
    if (mine) run_begin = found;
    wanted &= ~__ballot(mine);
  }
  // The first block that begins in the piece: of that run, or where it ends before that.
  const int done = (int)(first - run_begin) & (s.run - 1);
  const long long next = done ? end - done : first;
  const bool ends_here = inside && key_at(next) != token;
  if (inside && !ends_here) place = begin = next, whole = false;
  for (unsigned long long wanted = __ballot(ends_here); wanted;) {
    const int lane = __builtin_ctzll(wanted), at = __builtin_amdgcn_readlane(piece, lane);
    const unsigned of = (unsigned)__builtin_amdgcn_readlane((int)token, lane), key = key_at((long long)at * s.run + (threadIdx.x & 63));
    const int rows = __builtin_ctzll(__ballot(key != of));  // (of the run in the piece, which has fewer than 64 places)
    const bool mine = piece == at;
    if (mine) place = begin = first + rows;
    if (mine) token = (unsigned)__builtin_amdgcn_readlane((int)key, rows);
    wanted &= ~__ballot(mine);
  }
  if (token >= V || left == 0) return;  // (rows without a token are the last ones)
  float sum[8] = {};
  unsigned owner = token;  // (whose sum this is)
  auto flush = [&](bool ends) {
    if (whole && ends) {
      embedding_put((AT*)a.out + owner * a.D + col, left, sum, a.scale);
    } else {
      Eight<float> q;
      q.set(sum);
      q.store((whole ? s.begun : s.rest) + piece * s.pitch + col);
    }
  };
  constexpr int AHEAD = 8;
  bool ends = false;
  for (bool done = false; !done; place += AHEAD) {
    Eight<AT> q[AHEAD];
    unsigned key[AHEAD + 1], row[AHEAD], taken = 0, begins = 0;
    float part[8];
#pragma unroll
    for (int p = 0; p <= AHEAD; ++p) {
      key[p] = key_at(place + p);
      if (p < AHEAD) row[p] = a.order[place + p < a.rows ? place + p : a.rows - 1];
    }
#pragma unroll
    for (int p = 0; p <= AHEAD; ++p) {
      const bool other = key[p] != token, over = other ? place + p >= end || key[p] >= V : place + p - begin == s.run;
      if (!done && over) done = true, ends = other;
      if (p < AHEAD && !done) {
        if (other) token = key[p], begin = place + p, begins |= 1u << p;
        taken |= 1u << p;
      }
    }
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      const AT* from = (const AT*)a.in + row[p] * a.ld + col;
      const bool wanted = taken >> p & 1;
      if (wanted && left == 8) {
        q[p].load(from);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) part[k] = wanted && k < left ? load_f32(from + k) : 0.f;
        q[p].set(part);
      }
    }
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      if (begins >> p & 1) {
        flush(true);
        owner = key[p], whole = true;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = 0.f;
      }
      if (taken >> p & 1) {
        q[p].get(part);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] += part[k];
      }
    }
  }
  flush(ends);
}

// Rows of the table that are the sum of several blocks: a wavefront for each piece and 512 columns, which adds the blocks of the run that begins in the piece and is longer than one, if there is one; most pieces have none.
// The blocks of one token are added one after the other, 16 on their way at a time: a token of very many rows takes longer than the others together (131072 rows of 512 bf16, forward and gradient: 122 us
// with no token frequent, 240 with half of the rows one token, 323 with all).
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding_join(EmbeddingSumArgs s) {
  const EmbeddingArgs& a = s.e;
  const int lane = threadIdx.x & 63;
  const long long item = blockIdx.x * 4ll + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int piece = (int)(item / s.strips), strip = (int)(item - (long long)piece * s.strips);
  const long long first = (long long)piece * s.run;
  if (first + s.run >= a.rows) return;
  // (a lane for each of the piece's places, and for as many behind them: of a run that begins at the piece's place n the next block begins n lanes behind the last one's)
  const unsigned key = a.token_of[first + lane < a.rows ? first + lane : a.rows - 1], token = (unsigned)__builtin_amdgcn_readlane((int)key, s.run - 1);
  const int at = __builtin_ctzll(__ballot(key == token));
  if (token >= (unsigned)a.V || (at == 0 && first && a.token_of[first - 1] == token)) return;
  const long long next = first + at + s.run;
  if (next >= a.rows || (unsigned)__builtin_amdgcn_readlane((int)key, at + s.run) != token) return;
  int count = 0;  // pieces behind this one that begin with the token
  for (;;) {
    const long long at = next + (long long)(count + lane) * s.run;
    const unsigned long long other = ~__ballot(at < a.rows && a.token_of[at < a.rows ? at : next] == token);
    if (other) {
      count += __builtin_ctzll(other);
      break;
    }
    count += 64;
  }
  const long long col = strip * 512ll + lane * 8;
  const int left = (int)(a.D - col < 0 ? 0 : (a.D - col < 8 ? a.D - col : 8));
  if (left == 0) return;
  // (all of them asked for before the first is added: left to itself the compiler may ask for each only then)
  constexpr int AHEAD = 16;
  Eight<float> q[AHEAD];
  float sum[8], part[8];
  q[0].load(s.begun + piece * s.pitch + col);
  q[0].get(sum);
  const float* from = s.rest + (piece + 1) * s.pitch + col;
  for (int p0 = 0; p0 < count; p0 += AHEAD) {
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) q[p].load(from + (p0 + p < count ? p0 + p : p0) * s.pitch);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
      q[p].get(part);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] = p0 + p < count ? sum[k] + part[k] : sum[k];
    }
  }
  embedding_put((AT*)a.out + token * a.D + col, left, sum, a.scale);
}

}  // namespace rtn
