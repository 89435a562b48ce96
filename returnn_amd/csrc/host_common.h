// What the host sides of the operators' libraries share: the text of the last error, checks of arguments, choices of types.  Included once per library.
#pragma once

#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <string>
#include <type_traits>

#include "../../include/rtn_native_lstm2.h" /* status codes and element types */

namespace rtn {
namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RTN_OK : fail(RTN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

bool known(int dtype) { return dtype == RTN_DTYPE_F32 || dtype == RTN_DTYPE_BF16; }
int size_of(int dtype) { return dtype == RTN_DTYPE_BF16 ? 2 : 4; }
bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }
// Workgroups of a launch: its threads are counted in 32 bits.
constexpr int64_t max_blocks(int64_t threads) { return 0xFFFFFFFFll / threads; }
constexpr int64_t kMaxRows = 0x7FFFFFFF;

// Calls f with a value of the element type.
template <typename F>
void with_type(int dtype, F f) {
  if (dtype == RTN_DTYPE_BF16)
    f((__bf16)0.f);
  else
    f(0.f);
}

// Calls f with std::true_type or std::false_type.
template <typename F>
void with_bool(bool v, F f) {
  if (v)
    f(std::true_type());
  else
    f(std::false_type());
}

}  // namespace
}  // namespace rtn
