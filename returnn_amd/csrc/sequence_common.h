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

// Frames of sequence b: its length, or all there are.
__device__ __forceinline__ long long frames_of(const int64_t* lens, int b, long long T) {
  if (!lens) return T;
  const long long l = lens[b];
  return l < 0 ? 0 : (l > T ? T : l);
}

}  // namespace rtn
