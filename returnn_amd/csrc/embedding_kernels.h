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

// Where a row comes when rows are ordered by their tokens: after all of lower tokens and the earlier ones of the same.  Rows without a token come last.
__global__ __launch_bounds__(256) void k_embedding_order(EmbeddingArgs a) {
  const long long r = blockIdx.x * 256ll + threadIdx.x;
  auto token = [&](long long i) {
    const long long t = a.tokens[i];
    return t < 0 || t >= a.V ? a.V : t;
  };
  if (r >= a.rows) return;
  const long long mine = token(r);
  unsigned before = 0;
  for (long long i = 0; i < a.rows; ++i) {
    const long long t = token(i);
    before += t < mine || (t == mine && i < r);
  }
  a.order[before] = (unsigned)r;
  a.token_of[before] = (unsigned)mine;
}

// One row of the table per workgroup.
template <typename AT>
__global__ __launch_bounds__(256) void k_embedding_grad(EmbeddingArgs a) {
  const unsigned v = blockIdx.x;
  unsigned lo = 0, hi = (unsigned)a.rows;
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    if (a.token_of[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  for (long long e = threadIdx.x; e < a.D; e += 256) {
    float sum = 0.f;
    for (unsigned p = lo; p < a.rows && a.token_of[p] == v; ++p) sum += load_f32((const AT*)a.in + a.order[p] * a.ld + e);
    store_f32((AT*)a.out + v * a.D + e, sum * a.scale);
  }
}

}  // namespace rtn
