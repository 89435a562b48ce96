// The torch side of librtn_sequence_ops.so: argument checks, outputs, autograd nodes and the calls of its C ABI on torch tensors.
//
// The library's entry points come in as addresses (init), so that the Python side decides which library is loaded.
#include "../../include/rtn_sequence_ops.h"
#include "torch_binding_common.h"

namespace {

struct Abi {
  decltype(&rtn_sequence_last_error) last_error;
  decltype(&rtn_gated_recurrence_saved_bytes) recurrence_saved_bytes;
  decltype(&rtn_gated_recurrence_fwd_workspace_bytes) recurrence_fwd_workspace_bytes;
  decltype(&rtn_gated_recurrence_fwd) recurrence_fwd;
  decltype(&rtn_gated_recurrence_bwd_workspace_bytes) recurrence_bwd_workspace_bytes;
  decltype(&rtn_gated_recurrence_bwd) recurrence_bwd;
  decltype(&rtn_dropout) dropout;
  decltype(&rtn_token_log_probs_workspace_bytes) scores_workspace_bytes;
  decltype(&rtn_token_log_probs_fwd) scores_fwd;
  decltype(&rtn_token_log_probs_bwd) scores_bwd;
} abi;

void check_rc(int rc) {
  if (rc == RTN_OK) return;
  const char* text = abi.last_error();
  TORCH_CHECK(false, (text && *text) ? std::string(text) : "sequence ops: error code " + std::to_string(rc));
}

// ---- gated recurrence -----------------------------------------------------------------------------------------------
struct Recurrence {
  Tensor y, c, saved;
};
// x [T,B,4n], c0 [B,n] float32 or undefined, lens [B] int64 on the device or undefined
Recurrence recurrence_forward(const Tensor& x_in, const Tensor& c0, const Tensor& lens, int64_t direction, bool keep) {
  int64_t ld;
  const Tensor x = rows_of(x_in, &ld);
  const int64_t T = x.size(0), B = x.size(1), n = x.size(2) / 4;
  const int dtype = dtype_of(x);
  c10::DeviceGuard guard(x.device());
  Recurrence r;
  r.y = fresh({T, B, n}, x);
  r.c = fresh({B, n}, at::kFloat, x);
  if (keep) r.saved = scratch(abi.recurrence_saved_bytes(T, (int)B, (int)n, dtype), x);
  const size_t bytes = abi.recurrence_fwd_workspace_bytes(T, (int)B, (int)n, dtype);
  const Tensor ws = scratch(bytes, x);
  check_rc(abi.recurrence_fwd(pointer(x), ld, (const float*)pointer(c0), (const int64_t*)pointer(lens), pointer(r.y), (float*)pointer(r.c), pointer(r.saved), T, (int)B, (int)n,
                              dtype, (int)direction, pointer(ws), bytes, current_stream(x.device())));
  return r;
}

struct RecurrenceFunction : torch::autograd::Function<RecurrenceFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& c0, const std::optional<Tensor>& lens, int64_t direction) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Recurrence r = recurrence_forward(x, c0.value_or(Tensor()), lens.value_or(Tensor()), direction, true);
    ctx->save_for_backward({x, lens.value_or(Tensor()), r.saved});
    ctx->saved_data["direction"] = direction;
    ctx->saved_data["state"] = c0.has_value();
    ctx->set_materialize_grads(false);
    return {r.y, r.c};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_recurrence");
    const auto saved = ctx->get_saved_variables();
    int64_t ld, ldd;
    const Tensor x = rows_of(saved[0], &ld), &lens = saved[1];
    const int64_t T = x.size(0), B = x.size(1), n = x.size(2) / 4;
    const int dtype = dtype_of(x);
    c10::DeviceGuard guard(x.device());
    const Tensor dy = rows_of(grads[0].defined() ? grads[0] : at::zeros({T, B, n}, x.options()), &ldd);
    const Tensor dc = grads[1].defined() ? packed(grads[1]) : Tensor();
    const Tensor dx = fresh({T, B, 4 * n}, x), dc0 = fresh({B, n}, at::kFloat, x);
    const size_t bytes = abi.recurrence_bwd_workspace_bytes(T, (int)B, (int)n, dtype);
    const Tensor ws = scratch(bytes, x);
    check_rc(abi.recurrence_bwd(pointer(x), ld, nullptr, (const int64_t*)pointer(lens), pointer(saved[2]), pointer(dy), ldd, (const float*)pointer(dc), pointer(dx),
                                (float*)pointer(dc0), T, (int)B, (int)n, dtype, (int)ctx->saved_data["direction"].toInt(), pointer(ws), bytes, current_stream(x.device())));
    return {dx, ctx->saved_data["state"].toBool() ? dc0 : Tensor(), Tensor(), Tensor()};  // (no gradient for what was not given)
  }
};

std::tuple<Tensor, Tensor> gated_recurrence(const Tensor& source, const std::optional<Tensor>& state, const std::optional<Tensor>& lens_in, int64_t direction) {
  const char* what = "gated_recurrence";
  const Tensor x_in = in_region(source);
  check_input(x_in, what);
  TORCH_CHECK(x_in.dim() == 2 || x_in.dim() == 3, what, ": the input must be [T,B,4n] or [B,4n], got ", x_in.sizes());
  TORCH_CHECK(x_in.size(-1) % 4 == 0, what, ": the last axis of the input holds four gates of one width, got ", x_in.sizes());
  TORCH_CHECK(direction == 1 || direction == -1, what, ": direction must be +1 or -1");
  const bool single = x_in.dim() == 2;
  const int64_t B = x_in.size(-2), n = x_in.size(-1) / 4;
  TORCH_CHECK(B <= INT_MAX && n <= INT_MAX / 4, what, ": input ", x_in.sizes(), " is too large");
  std::optional<Tensor> c0, lens;
  if (state.has_value()) {
    TORCH_CHECK(state->sizes() == at::IntArrayRef({B, n}), what, ": state ", state->sizes(), ", expected ", at::IntArrayRef({B, n}));
    same_device(*state, x_in, what, "the state");
    no_tangent(*state, what);
    TORCH_CHECK(at::isFloatingType(state->scalar_type()), what, ": state of type ", state->scalar_type());
    c0 = packed(as_type(*state, at::kFloat));
  }
  if (lens_in.has_value()) {
    TORCH_CHECK(lens_in->sizes() == at::IntArrayRef({B}), what, ": seq_lens ", lens_in->sizes(), ", expected ", at::IntArrayRef({B}));
    TORCH_CHECK(at::isIntegralType(lens_in->scalar_type(), false), what, ": seq_lens of type ", lens_in->scalar_type());
    lens = packed(as_type(lens_in->to(x_in.device()), at::kLong));
  }
  const Tensor x = single ? x_in.unsqueeze(0) : x_in;
  Tensor y, c;
  if (at::GradMode::is_enabled() && (x.requires_grad() || (c0.has_value() && c0->requires_grad()))) {
    const variable_list r = RecurrenceFunction::apply(x, c0, lens, direction);
    y = r[0], c = r[1];
  } else {
    const Recurrence r = recurrence_forward(x, c0.value_or(Tensor()), lens.value_or(Tensor()), direction, false);
    y = r.y, c = r.c;
  }
  return {single ? y.squeeze(0) : y, c};
}

// ---- dropout --------------------------------------------------------------------------------------------------------
struct DropoutKey {
  int64_t threshold;
  uint64_t seed, offset;
  bool same_over_time;
};
Tensor dropout_call(const Tensor& x_in, const Tensor& residual_in, const Tensor& offset, const DropoutKey& key) {
  // (What lies in one piece is one row, whatever its width.)
  Tensor x = x_in.dim() == 1 ? packed(x_in) : x_in, residual = residual_in;
  if (x.dim() == 1 && residual.defined()) residual = packed(residual);
  const int64_t outer = key.same_over_time ? x.size(0) : 1;
  const bool flat = x.is_contiguous() && (!residual.defined() || residual.is_contiguous());
  int64_t times = outer, rows = 1, width = x.numel() / std::max<int64_t>(outer, 1), ldx = width, ldr = width;
  if (!flat) {
    width = x.size(-1);
    rows = x.numel() / std::max<int64_t>(outer * width, 1);
    x = rows_of(x, &ldx);
    if (residual.defined()) residual = rows_of(residual, &ldr);
  }
  c10::DeviceGuard guard(x.device());
  const Tensor y = fresh(x.sizes(), x);
  if (y.numel())
    check_rc(abi.dropout(pointer(x), ldx, pointer(residual), ldr, pointer(y), times, rows, width, dtype_of(x), (int)key.threshold, key.seed, key.offset,
                         (const int64_t*)pointer(offset), key.same_over_time, current_stream(x.device())));
  return y;
}

struct DropoutFunction : torch::autograd::Function<DropoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual, const std::optional<Tensor>& offset, int64_t threshold, int64_t seed,
                        int64_t base, bool same_over_time) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({offset.value_or(Tensor())});
    ctx->saved_data["threshold"] = threshold;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["base"] = base;
    ctx->saved_data["same"] = same_over_time;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_call(x, residual.value_or(Tensor()), offset.value_or(Tensor()), {threshold, (uint64_t)seed, (uint64_t)base, same_over_time});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("dropout");
    variable_list out(7);
    const DropoutKey key{ctx->saved_data["threshold"].toInt(), (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["base"].toInt(),
                         ctx->saved_data["same"].toBool()};
    if (ctx->needs_input_grad(0)) out[0] = dropout_call(grads[0], Tensor(), ctx->get_saved_variables()[0], key);
    if (ctx->saved_data["residual"].toBool()) out[1] = grads[0];
    return out;
  }
};

Tensor dropout(const Tensor& source, int64_t threshold, uint64_t seed, uint64_t base, const std::optional<Tensor>& offset, const std::optional<Tensor>& residual_in,
               bool same_over_time) {
  const char* what = "dropout";
  const Tensor x = in_region(source);
  std::optional<Tensor> residual;
  if (residual_in.has_value()) residual = in_region(*residual_in);
  check_input(x, what);
  TORCH_CHECK(x.dim() >= 1, what, ": the input has no axis");
  if (residual.has_value()) {
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(), what, ": residual ", residual->sizes(), " of ", residual->scalar_type(),
                ", expected ", x.sizes(), " of ", x.scalar_type());
    same_device(*residual, x, what, "the residual");
    no_tangent(*residual, what);
  }
  if (offset.has_value()) {
    TORCH_CHECK(offset->scalar_type() == at::kLong && offset->numel() == 1, what, ": an offset on the device is one int64, got ", offset->sizes(), " of ", offset->scalar_type());
    same_device(*offset, x, what, "the offset");
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || (residual.has_value() && residual->requires_grad())))
    return DropoutFunction::apply(x, residual, offset, threshold, (int64_t)seed, (int64_t)base, same_over_time);
  return dropout_call(x, residual.value_or(Tensor()), offset.value_or(Tensor()), {threshold, seed, base, same_over_time});
}

// ---- scores of tokens -----------------------------------------------------------------------------------------------
struct Scores {
  Tensor log_prob, entropy, top_log_prob, top_ids, norm;
};
Scores scores_forward(const Tensor& logits_in, const Tensor& targets, bool entropy, int64_t top_k, bool keep) {
  int64_t ld;
  const Tensor logits = rows_of(logits_in, &ld);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const int64_t V = logits.size(-1), rows = c10::multiply_integers(lead);
  const int dtype = dtype_of(logits);
  c10::DeviceGuard guard(logits.device());
  Scores s;
  if (targets.defined()) s.log_prob = fresh(lead, at::kFloat, logits);
  if (entropy) s.entropy = fresh(lead, at::kFloat, logits);
  std::vector<int64_t> alternatives(lead.begin(), lead.end());
  alternatives.push_back(top_k);
  s.top_log_prob = fresh(alternatives, at::kFloat, logits);
  s.top_ids = fresh(alternatives, at::kLong, logits);
  if (keep) s.norm = fresh({rows, 2}, at::kFloat, logits);
  const size_t bytes = abi.scores_workspace_bytes(rows, V, dtype, (int)top_k);
  const Tensor ws = scratch(bytes, logits);
  check_rc(abi.scores_fwd(pointer(logits), ld, (const int64_t*)pointer(targets), rows, V, dtype, (int)top_k, (float*)pointer(s.log_prob), (float*)pointer(s.norm),
                          (float*)pointer(s.entropy), (float*)pointer(s.top_log_prob), (int64_t*)pointer(s.top_ids), pointer(ws), bytes, current_stream(logits.device())));
  return s;
}

struct ScoresFunction : torch::autograd::Function<ScoresFunction> {
  // (log_prob, entropy, top_log_prob, top_ids), those not wanted left out of the front: as `has` says
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const std::optional<Tensor>& targets, bool entropy, int64_t top_k) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Scores s = scores_forward(logits, targets.value_or(Tensor()), entropy, top_k, true);
    ctx->save_for_backward({logits, targets.value_or(Tensor()), s.norm, entropy ? s.entropy : Tensor()});
    ctx->mark_non_differentiable({s.top_log_prob, s.top_ids});
    ctx->set_materialize_grads(false);
    variable_list out;
    if (targets.has_value()) out.push_back(s.log_prob);
    if (entropy) out.push_back(s.entropy);
    out.push_back(s.top_log_prob);
    out.push_back(s.top_ids);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("token_log_probs");
    const auto saved = ctx->get_saved_variables();
    int64_t ld;
    const Tensor logits = rows_of(saved[0], &ld), &targets = saved[1], &norm = saved[2], &entropy = saved[3];
    size_t at_grad = 0;
    const Tensor g = targets.defined() ? grads[at_grad++] : Tensor(), ge = entropy.defined() ? grads[at_grad++] : Tensor();
    c10::DeviceGuard guard(logits.device());
    const Tensor g1 = g.defined() ? packed(g) : Tensor(), g2 = ge.defined() ? packed(ge) : Tensor();
    const Tensor D = fresh(logits.sizes(), logits);
    const int64_t V = logits.size(-1), rows = norm.size(0);
    check_rc(abi.scores_bwd(pointer(logits), ld, (const int64_t*)pointer(targets), (const float*)pointer(norm), (const float*)pointer(entropy), (const float*)pointer(g1),
                            (const float*)pointer(g2), pointer(D), rows, V, dtype_of(logits), current_stream(logits.device())));
    return {D, Tensor(), Tensor(), Tensor()};
  }
};

// (log_probs or None, entropy or None, top_log_probs, top_ids)
py::tuple token_log_probs(const Tensor& logits_in, const std::optional<Tensor>& targets_in, bool entropy, int64_t top_k) {
  const char* what = "token_log_probs";
  const Tensor logits = in_region(logits_in);
  check_input(logits, what);
  TORCH_CHECK(logits.dim() >= 1 && logits.size(-1) > 0, what, ": logits ", logits.sizes(), " have no tokens");
  TORCH_CHECK(top_k >= 0 && top_k <= 64 && top_k <= logits.size(-1), what, ": top_k must be in 0..", std::min<int64_t>(64, logits.size(-1)), ", got ", top_k);
  std::optional<Tensor> targets;
  if (targets_in.has_value()) {
    TORCH_CHECK(targets_in->sizes() == logits.sizes().slice(0, logits.dim() - 1), what, ": targets ", targets_in->sizes(), " do not match logits ", logits.sizes());
    TORCH_CHECK(at::isIntegralType(targets_in->scalar_type(), false), what, ": targets of type ", targets_in->scalar_type());
    same_device(*targets_in, logits, what, "a target");
    targets = packed(as_type(*targets_in, at::kLong));
  }
  py::object log_probs = py::none(), h = py::none();
  if (at::GradMode::is_enabled() && logits.requires_grad() && (targets.has_value() || entropy)) {
    const variable_list r = ScoresFunction::apply(logits, targets, entropy, top_k);
    size_t k = 0;
    if (targets.has_value()) log_probs = py::cast(r[k++]);
    if (entropy) h = py::cast(r[k++]);
    return py::make_tuple(log_probs, h, r[k], r[k + 1]);
  }
  const Scores s = scores_forward(logits, targets.value_or(Tensor()), entropy, top_k, false);
  if (targets.has_value()) log_probs = py::cast(s.log_prob);
  if (entropy) h = py::cast(s.entropy);
  return py::make_tuple(log_probs, h, s.top_log_prob, s.top_ids);
}

void init(const py::dict& symbols) {
  take(abi.last_error, symbols, "rtn_sequence_last_error");
  take(abi.recurrence_saved_bytes, symbols, "rtn_gated_recurrence_saved_bytes");
  take(abi.recurrence_fwd_workspace_bytes, symbols, "rtn_gated_recurrence_fwd_workspace_bytes");
  take(abi.recurrence_fwd, symbols, "rtn_gated_recurrence_fwd");
  take(abi.recurrence_bwd_workspace_bytes, symbols, "rtn_gated_recurrence_bwd_workspace_bytes");
  take(abi.recurrence_bwd, symbols, "rtn_gated_recurrence_bwd");
  take(abi.dropout, symbols, "rtn_dropout");
  take(abi.scores_workspace_bytes, symbols, "rtn_token_log_probs_workspace_bytes");
  take(abi.scores_fwd, symbols, "rtn_token_log_probs_fwd");
  take(abi.scores_bwd, symbols, "rtn_token_log_probs_bwd");
  ready = true;
}

}  // namespace

PYBIND11_MODULE(_rtn_sequence, m) {
  m.def("init", &init);
  m.def("gated_recurrence", &gated_recurrence);
  m.def("dropout", &dropout);
  m.def("token_log_probs", &token_log_probs);
}
