// What the torch sides of the operators' libraries share: checks, types, outputs, rows with a pitch.  Included once per binding.
#pragma once

#include <torch/extension.h>

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <string>
#include <vector>

#include "../../include/rtn_native_lstm2.h" /* status codes and element types */

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

bool ready = false;  // (whether the library's entry points are known)

hipStream_t current_stream(const at::Device& device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

// The ops have a gradient, but none in forward mode: a tangent would be lost.
void no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, ": derivatives in forward mode are not implemented for this op");
}

// What every op wants of its main input.
void check_input(const Tensor& t, const char* what) {
  TORCH_CHECK(ready, what, ": the library is not loaded");
  TORCH_CHECK(t.is_cuda(), what, ": this build implements the op for HIP (MI355X) tensors only; got a CPU tensor");
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, what, ": float32 or bfloat16 needed, got ", t.scalar_type());
  no_tangent(t, what);
}
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RTN_DTYPE_BF16 : RTN_DTYPE_F32; }
void same_device(const Tensor& t, const Tensor& as, const char* what, const char* name) {
  TORCH_CHECK(t.device() == as.device(), what, ": ", name, " is on ", t.device(), " but the input is on ", as.device());
}
Tensor as_type(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }
// (a view that says of itself that its numbers are to be negated or conjugated is made what it says first)
Tensor resolved(const Tensor& t) { return t.is_neg() || t.is_conj() ? t.resolve_conj().resolve_neg() : t; }
Tensor packed(const Tensor& t) { return resolved(t).contiguous(); }
void* pointer(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
// (not through the dispatcher: host time of the alternatives of 12 rows 5.6 us with it, 5.0 without)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
Tensor fresh(at::IntArrayRef sizes, const Tensor& like) { return fresh(sizes, like.scalar_type(), like); }
Tensor scratch(size_t bytes, const Tensor& like) { return bytes ? fresh({(int64_t)bytes}, at::kByte, like) : Tensor(); }

// What a matrix product of an autocast region gives, as these ops take it: as for the LSTM layers bfloat16 where that is the region's type, else float32.  (The cast
// is one that autograd sees.)  Outside a region float16 is refused.
Tensor in_region(const Tensor& t) {
  return t.scalar_type() == at::kHalf && t.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA) ? t.to(at::kFloat) : t;
}

// Elements from one row to the next where a row is what the last axis holds and the rows, in order, are equally far apart; 0 where they are not.
int64_t row_pitch(const Tensor& t) {
  const int64_t width = t.size(-1);
  if (t.numel() == 0) return width;
  if (width > 1 && t.stride(-1) != 1) return 0;
  int64_t pitch = -1, next = 0;  // (next: what the stride of the next axis outwards has to be)
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (pitch < 0)
      pitch = t.stride(d);
    else if (t.stride(d) != next)
      return 0;
    if (pitch < width) return 0;  // (rows that overlap, such as those of an expanded tensor)
    next = t.stride(d) * t.size(d);
  }
  return pitch < 0 ? width : pitch;
}
// t as it can be handed over, and its pitch.
Tensor rows_of(const Tensor& view, int64_t* pitch) {
  const Tensor t = resolved(view);
  if ((*pitch = row_pitch(t))) return t;
  *pitch = t.size(-1);
  return t.contiguous();
}

void once(const char* what) { TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient has no gradient of its own (create_graph=True)"); }

template <typename F>
void take(F*& fn, const py::dict& symbols, const char* name) {
  fn = reinterpret_cast<F*>(symbols[name].cast<uintptr_t>());
}

}  // namespace
