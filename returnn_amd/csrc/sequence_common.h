// What the kernels of the sequence operators share: element types and small helpers.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace rtn {

template <typename AT>
__device__ __forceinline__ float load_f32(const AT* p) {
  return (float)*p;
}
template <typename AT>
__device__ __forceinline__ void store_f32(AT* p, float v) {  // rounds to nearest, ties to even
  *p = (AT)v;
}

// Two numbers rounded to bfloat16, the first in the lower half.
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  typedef __attribute__((__vector_size__(2 * sizeof(float)))) float pair_f32;
  typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 pair_bf16;
  return __builtin_bit_cast(unsigned, __builtin_convertvector((pair_f32){a, b}, pair_bf16));
}

// Eight neighbouring elements as they lie in memory, at any element's address: one load of 16 bytes in bfloat16, two in float32 (the
// hardware takes them at any address).
typedef __attribute__((__vector_size__(4 * sizeof(unsigned)))) unsigned seq_u32x4;
typedef seq_u32x4 __attribute__((aligned(2))) seq_u32x4_any;
template <typename AT>
struct Eight {
  static constexpr int kWords = sizeof(AT) == 2 ? 1 : 2;
  seq_u32x4 w[kWords];
  __device__ __forceinline__ void load(const AT* p) {
#pragma unroll
    for (int j = 0; j < kWords; ++j) w[j] = ((const seq_u32x4_any*)p)[j];
  }
  __device__ __forceinline__ void store(AT* p) const {
#pragma unroll
    for (int j = 0; j < kWords; ++j) ((seq_u32x4_any*)p)[j] = w[j];
  }
  __device__ __forceinline__ void store_streamed(AT* p) const {  // of what is not read again before much else is
#pragma unroll
    for (int j = 0; j < kWords; ++j) __builtin_nontemporal_store(w[j], (seq_u32x4_any*)p + j);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if constexpr (sizeof(AT) == 2)
        v[k] = __builtin_bit_cast(float, k & 1 ? w[0][k >> 1] & 0xFFFF0000u : w[0][k >> 1] << 16);
      else
        v[k] = __builtin_bit_cast(float, (unsigned)w[k >> 2][k & 3]);  // (without the cast the compiler takes the first word for all)
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if constexpr (sizeof(AT) == 4) w[k >> 2][k & 3] = __builtin_bit_cast(unsigned, v[k]);
    if constexpr (sizeof(AT) == 2) {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[0][k] = pack_bf16(v[2 * k], v[2 * k + 1]);
    }
  }
};

// Frames of sequence b: its length, or all there are.
__device__ __forceinline__ long long frames_of(const int64_t* lens, int b, long long T) {
  if (!lens) return T;
  const long long l = lens[b];
  return l < 0 ? 0 : (l > T ? T : l);
}

}  // namespace rtn
