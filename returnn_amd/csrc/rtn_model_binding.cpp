// The torch side of librtn_model_ops.so: argument checks, outputs, autograd nodes and the calls of its C ABI on torch tensors.
//
// The library's entry points come in as addresses (init), so that the Python side decides which library is loaded.
#include "../../include/rtn_model_ops.h"
#include "torch_binding_common.h"

namespace {

struct Abi {
  decltype(&rtn_model_ops_last_error) last_error;
  decltype(&rtn_delta_rule_fwd_workspace_bytes) delta_fwd_workspace_bytes;
  decltype(&rtn_delta_rule_saved_bytes) delta_saved_bytes;
  decltype(&rtn_delta_rule_fwd) delta_fwd;
  decltype(&rtn_delta_rule_bwd_workspace_bytes) delta_bwd_workspace_bytes;
  decltype(&rtn_delta_rule_bwd) delta_bwd;
  decltype(&rtn_embedding_fwd) embedding_fwd;
  decltype(&rtn_embedding_bwd_workspace_bytes) embedding_bwd_workspace_bytes;
  decltype(&rtn_embedding_bwd) embedding_bwd;
  decltype(&rtn_beam_select_workspace_bytes) beam_workspace_bytes;
  decltype(&rtn_beam_select) beam_select;
  decltype(&rtn_reorder_rows) reorder_rows;
} abi;

void check_rc(int rc) {
  if (rc == RTN_OK) return;
  const char* text = abi.last_error();
  TORCH_CHECK(false, (text && *text) ? std::string(text) : "model ops: error code " + std::to_string(rc));
}

// ---- gated delta rule -----------------------------------------------------------------------------------------------
struct DeltaSizes {
  int64_t T;
  int B, key_heads, heads, dk, dv, dtype;
};
DeltaSizes delta_sizes(const Tensor& q, const Tensor& v) {
  return {v.size(0), (int)v.size(1), (int)q.size(2), (int)v.size(2), (int)q.size(3), (int)v.size(3), dtype_of(v)};
}
// [T,B,heads,width] as rows of all heads.
Tensor head_rows(const Tensor& t, int64_t* pitch) { return rows_of(t.flatten(2), pitch); }

struct Delta {
  Tensor y, s, saved;
};
// q, k [T,B,key_heads,dk], v [T,B,heads,dv], g, beta [T,B,heads] float32; s0 [B,heads,dk,dv] float32 or undefined; lens [B] int64 on the device or undefined
Delta delta_forward(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& g, const Tensor& beta, const Tensor& s0, const Tensor& lens, double scale,
                    int64_t direction, bool keep) {
  const DeltaSizes z = delta_sizes(q_in, v_in);
  int64_t ldq, ldk, ldv;
  c10::DeviceGuard guard(v_in.device());
  const Tensor q = head_rows(q_in, &ldq), k = head_rows(k_in, &ldk), v = head_rows(v_in, &ldv);
  Delta r;
  r.y = fresh(v_in.sizes(), v);
  r.s = fresh({z.B, z.heads, z.dk, z.dv}, at::kFloat, v);
  if (keep) r.saved = scratch(abi.delta_saved_bytes(z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, z.dtype), v);
  const size_t bytes = abi.delta_fwd_workspace_bytes(z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, z.dtype, keep);
  const Tensor ws = scratch(bytes, v);
  check_rc(abi.delta_fwd(pointer(q), ldq, pointer(k), ldk, pointer(v), ldv, (const float*)pointer(g), (const float*)pointer(beta), (const float*)pointer(s0),
                         (const int64_t*)pointer(lens), pointer(r.y), (float*)pointer(r.s), pointer(r.saved), z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, z.dtype, (float)scale,
                         (int)direction, pointer(ws), bytes, current_stream(v.device())));
  return r;
}

struct DeltaFunction : torch::autograd::Function<DeltaFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta, const std::optional<Tensor>& s0,
                               const std::optional<Tensor>& lens, double scale, int64_t direction) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Delta r = delta_forward(q, k, v, g, beta, s0.value_or(Tensor()), lens.value_or(Tensor()), scale, direction, true);
    ctx->save_for_backward({q, k, v, g, beta, lens.value_or(Tensor()), r.saved});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["direction"] = direction;
    ctx->saved_data["state"] = s0.has_value();
    ctx->set_materialize_grads(false);
    return {r.y, r.s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_delta_rule");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q_in = saved[0], &k_in = saved[1], &v_in = saved[2], &g = saved[3], &beta = saved[4], &lens = saved[5];
    const DeltaSizes z = delta_sizes(q_in, v_in);
    int64_t ldq, ldk, ldv, ldy;
    c10::DeviceGuard guard(v_in.device());
    const Tensor q = head_rows(q_in, &ldq), k = head_rows(k_in, &ldk), v = head_rows(v_in, &ldv);
    const Tensor dy = head_rows(grads[0].defined() ? grads[0] : at::zeros(v_in.sizes(), v_in.options()), &ldy);
    const Tensor ds = grads[1].defined() ? packed(grads[1]) : Tensor();
    const Tensor dq = fresh(q_in.sizes(), q), dk = fresh(k_in.sizes(), k), dv = fresh(v_in.sizes(), v), dg = fresh(g.sizes(), g), db = fresh(g.sizes(), g);
    const Tensor ds0 = fresh({z.B, z.heads, z.dk, z.dv}, g);
    const size_t bytes = abi.delta_bwd_workspace_bytes(z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, z.dtype);
    const Tensor ws = scratch(bytes, v);
    check_rc(abi.delta_bwd(pointer(q), ldq, pointer(k), ldk, pointer(v), ldv, (const float*)pointer(g), (const float*)pointer(beta), (const int64_t*)pointer(lens),
                           pointer(saved[6]), pointer(dy), ldy, (const float*)pointer(ds), pointer(dq), pointer(dk), pointer(dv), (float*)pointer(dg), (float*)pointer(db),
                           (float*)pointer(ds0), z.T, z.B, z.key_heads, z.heads, z.dk, z.dv, z.dtype, (float)ctx->saved_data["scale"].toDouble(),
                           (int)ctx->saved_data["direction"].toInt(), pointer(ws), bytes, current_stream(v.device())));
    return {dq, dk, dv, dg, db, ctx->saved_data["state"].toBool() ? ds0 : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_delta_rule(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& decay_in, const Tensor& beta_in,
                                            const std::optional<double>& scale_in, const std::optional<Tensor>& state, const std::optional<Tensor>& lens_in, int64_t direction) {
  const char* what = "gated_delta_rule";
  Tensor q = in_region(query), k = in_region(key), v = in_region(value);
  check_input(v, what);
  TORCH_CHECK(v.dim() == 3 || v.dim() == 4, what, ": values must be [T,B,heads,dv] or [B,heads,dv], got ", v.sizes());
  TORCH_CHECK(q.dim() == v.dim() && k.sizes() == q.sizes() && q.sizes().slice(0, v.dim() - 2) == v.sizes().slice(0, v.dim() - 2), what, ": queries ", q.sizes(), " and keys ",
              k.sizes(), " do not match values ", v.sizes());
  TORCH_CHECK(q.scalar_type() == v.scalar_type() && k.scalar_type() == v.scalar_type(), what, ": queries, keys and values of one type needed, got ", q.scalar_type(), ", ",
              k.scalar_type(), ", ", v.scalar_type());
  const bool single = v.dim() == 3;
  const int64_t B = v.size(-3), H = v.size(-2), Hk = q.size(-2), dk = q.size(-1), dv = v.size(-1);
  TORCH_CHECK(Hk ? H % Hk == 0 : H == 0, what, ": ", H, " heads of values cannot share ", Hk, " heads of queries and keys evenly");
  TORCH_CHECK(dk >= 1 && dk <= 128 && dv >= 1 && dv <= 65536, what, ": keys of 1 to 128 and values of 1 to 65536 elements needed, got ", dk, " and ", dv);
  TORCH_CHECK(B <= INT_MAX && H <= INT_MAX && Hk <= INT_MAX, what, ": queries ", q.sizes(), " and values ", v.sizes(), " are too large");
  TORCH_CHECK(direction == 1 || direction == -1, what, ": direction must be +1 or -1");
  auto of_heads = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.sizes() == v.sizes().slice(0, v.dim() - 1), what, ": ", name, " ", t.sizes(), ", expected ", v.sizes().slice(0, v.dim() - 1));
    TORCH_CHECK(at::isFloatingType(t.scalar_type()), what, ": ", name, " of type ", t.scalar_type());
    return packed(as_type(t, at::kFloat));
  };
  auto beside = [&](const Tensor& t, const char* name) {
    same_device(t, v, what, name);
    no_tangent(t, what);
  };
  beside(q, "the queries"), beside(k, "the keys"), beside(decay_in, "log_decay"), beside(beta_in, "beta");
  Tensor g = of_heads(decay_in, "log_decay"), beta = of_heads(beta_in, "beta");
  std::optional<Tensor> s0, lens;
  if (state.has_value()) {
    TORCH_CHECK(state->sizes() == at::IntArrayRef({B, H, dk, dv}), what, ": state ", state->sizes(), ", expected ", at::IntArrayRef({B, H, dk, dv}));
    same_device(*state, v, what, "the state");
    no_tangent(*state, what);
    TORCH_CHECK(at::isFloatingType(state->scalar_type()), what, ": state of type ", state->scalar_type());
    s0 = packed(as_type(*state, at::kFloat));
  }
  if (lens_in.has_value()) {
    TORCH_CHECK(lens_in->sizes() == at::IntArrayRef({B}), what, ": seq_lens ", lens_in->sizes(), ", expected ", at::IntArrayRef({B}));
    TORCH_CHECK(at::isIntegralType(lens_in->scalar_type(), false), what, ": seq_lens of type ", lens_in->scalar_type());
    lens = packed(as_type(lens_in->to(v.device()), at::kLong));
  }
  const double scale = scale_in.value_or(1.0 / std::sqrt((double)dk));
  if (single) q = q.unsqueeze(0), k = k.unsqueeze(0), v = v.unsqueeze(0), g = g.unsqueeze(0), beta = beta.unsqueeze(0);
  Delta r;
  const bool wanted = q.requires_grad() || k.requires_grad() || v.requires_grad() || g.requires_grad() || beta.requires_grad() || (s0.has_value() && s0->requires_grad());
  if (at::GradMode::is_enabled() && wanted) {
    const variable_list out = DeltaFunction::apply(q, k, v, g, beta, s0, lens, scale, direction);
    r.y = out[0], r.s = out[1];
  } else {
    r = delta_forward(q, k, v, g, beta, s0.value_or(Tensor()), lens.value_or(Tensor()), scale, direction, false);
  }
  return {single ? r.y.squeeze(0) : r.y, r.s};
}

// ---- embedding ------------------------------------------------------------------------------------------------------
Tensor embedding_forward(const Tensor& tokens, const Tensor& table_in, double scale) {
  int64_t ld;
  const Tensor table = rows_of(table_in, &ld);
  c10::DeviceGuard guard(table.device());
  std::vector<int64_t> sizes(tokens.sizes().begin(), tokens.sizes().end());
  sizes.push_back(table.size(1));
  const Tensor y = fresh(sizes, table);
  check_rc(abi.embedding_fwd((const int64_t*)pointer(tokens), pointer(table), ld, pointer(y), tokens.numel(), table.size(0), table.size(1), dtype_of(table), (float)scale,
                             current_stream(table.device())));
  return y;
}

struct EmbeddingFunction : torch::autograd::Function<EmbeddingFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& table, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({tokens});
    ctx->saved_data["V"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    return embedding_forward(tokens, table, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("embed");
    const Tensor tokens = ctx->get_saved_variables()[0];
    int64_t ld;
    const Tensor dy = rows_of(grads[0], &ld);
    const int64_t V = ctx->saved_data["V"].toInt(), D = dy.size(-1), rows = tokens.numel();
    c10::DeviceGuard guard(dy.device());
    const Tensor d = fresh({V, D}, dy);
    const size_t bytes = abi.embedding_bwd_workspace_bytes(rows, V, D, dtype_of(dy));
    const Tensor ws = scratch(bytes, dy);
    check_rc(abi.embedding_bwd((const int64_t*)pointer(tokens), pointer(dy), ld, pointer(d), rows, V, D, dtype_of(dy), (float)ctx->saved_data["scale"].toDouble(), pointer(ws), bytes,
                               current_stream(dy.device())));
    return {Tensor(), d, Tensor()};
  }
};

Tensor embed(const Tensor& tokens_in, const Tensor& table_in, double scale) {
  const char* what = "embed";
  const Tensor table = in_region(table_in);
  check_input(table, what);
  TORCH_CHECK(table.dim() == 2, what, ": the table must be [V,D], got ", table.sizes());
  TORCH_CHECK(at::isIntegralType(tokens_in.scalar_type(), false), what, ": tokens of type ", tokens_in.scalar_type());
  same_device(tokens_in, table, what, "a token");
  const Tensor tokens = packed(as_type(tokens_in, at::kLong));
  if (at::GradMode::is_enabled() && table.requires_grad()) return EmbeddingFunction::apply(tokens, table, scale);
  return embedding_forward(tokens, table, scale);
}

// ---- beam search ----------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& scores_in, const Tensor& totals_in, int64_t beam, const std::optional<Tensor>& ended_in,
                                               const std::optional<int64_t>& end_token) {
  const char* what = "beam_select";
  const Tensor scores0 = in_region(scores_in);
  check_input(scores0, what);
  TORCH_CHECK(scores0.dim() == 2 || scores0.dim() == 3, what, ": scores must be [B,K,V] or [K,V], got ", scores0.sizes());
  const bool single = scores0.dim() == 2;
  const int64_t K = scores0.size(-2), V = scores0.size(-1), B = single ? 1 : scores0.size(0);
  const auto lead = scores0.sizes().slice(0, scores0.dim() - 1);
  TORCH_CHECK(K >= 1 && V >= 1 && V <= 1 << 26 && V <= INT_MAX / K && B <= INT_MAX, what, ": scores ", scores0.sizes(), ", up to 2^26 of a hypothesis and from 1 to 2^31 - 1 of a search needed");
  TORCH_CHECK(beam >= 1 && beam <= 64 && beam <= K * V, what, ": beam must be in 1..", std::min<int64_t>(64, K * V), ", got ", beam);
  TORCH_CHECK(totals_in.sizes() == lead, what, ": totals ", totals_in.sizes(), ", expected ", lead);
  TORCH_CHECK(totals_in.scalar_type() == at::kFloat, what, ": totals of type ", totals_in.scalar_type(), ", float32 needed");
  same_device(totals_in, scores0, what, "a total");
  no_tangent(totals_in, what);
  Tensor ended;
  if (ended_in.has_value()) {
    TORCH_CHECK(ended_in->sizes() == lead, what, ": ended ", ended_in->sizes(), ", expected ", lead);
    TORCH_CHECK(ended_in->scalar_type() == at::kBool, what, ": ended of type ", ended_in->scalar_type(), ", truth values needed");
    TORCH_CHECK(end_token.has_value() && *end_token >= 0 && *end_token < V, what, ": hypotheses that have ended need an end_token in 0..", V - 1);
    same_device(*ended_in, scores0, what, "ended");
    ended = packed(*ended_in);
  }
  int64_t ld;
  c10::DeviceGuard guard(scores0.device());
  const Tensor scores = rows_of(scores0.detach(), &ld), totals = packed(totals_in.detach());
  std::vector<int64_t> sizes;
  if (!single) sizes.push_back(B);
  sizes.push_back(beam);
  const Tensor out = fresh(sizes, at::kFloat, scores), sources = fresh(sizes, at::kLong, scores), tokens = fresh(sizes, at::kLong, scores);
  const size_t bytes = abi.beam_workspace_bytes((int)B, (int)K, V, dtype_of(scores), (int)beam);
  const Tensor ws = scratch(bytes, scores);
  check_rc(abi.beam_select(pointer(scores), ld, (const float*)pointer(totals), (const uint8_t*)pointer(ended), end_token.value_or(0), (float*)pointer(out),
                           (int64_t*)pointer(sources), (int64_t*)pointer(tokens), (int)B, (int)K, V, dtype_of(scores), (int)beam, pointer(ws), bytes,
                           current_stream(scores.device())));
  return {out, sources, tokens};
}

std::vector<Tensor> reorder_states(const std::vector<Tensor>& states, const Tensor& sources_in) {
  const char* what = "reorder_states";
  TORCH_CHECK(ready, what, ": the library is not loaded");
  TORCH_CHECK(sources_in.is_cuda(), what, ": this build implements the op for HIP (MI355X) tensors only; got a CPU tensor");
  TORCH_CHECK(sources_in.dim() == 1 || sources_in.dim() == 2, what, ": sources must be [B,beam] or [beam], got ", sources_in.sizes());
  TORCH_CHECK(sources_in.scalar_type() == at::kLong, what, ": sources of type ", sources_in.scalar_type(), ", int64 needed");
  const int64_t lead = sources_in.dim(), B = lead == 2 ? sources_in.size(0) : 1, beam = sources_in.size(-1);
  TORCH_CHECK(B <= INT_MAX && beam <= INT_MAX, what, ": sources ", sources_in.sizes(), " are too large");
  c10::DeviceGuard guard(sources_in.device());
  const Tensor sources = packed(sources_in);
  std::vector<Tensor> in, out;
  std::vector<const void*> from;
  std::vector<void*> to;
  std::vector<int64_t> bytes;
  int64_t K = -1;
  for (const Tensor& t : states) {
    TORCH_CHECK(t.dim() >= lead && (lead == 1 || t.size(0) == B), what, ": state ", t.sizes(), " does not begin with ", lead == 2 ? "[B,K]" : "[K]", " of sources ",
                sources_in.sizes());
    same_device(t, sources, what, "a state");
    no_tangent(t, what);
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, ": a state that requires a gradient; the op has none");
    if (K < 0) K = t.size(lead - 1);
    TORCH_CHECK(t.size(lead - 1) == K && K <= INT_MAX, what, ": states of ", K, " and of ", t.size(lead - 1), " hypotheses");
    in.push_back(packed(t));
    std::vector<int64_t> sizes(t.sizes().begin(), t.sizes().end());
    sizes[lead - 1] = beam;
    out.push_back(fresh(sizes, t));
    const int64_t row = c10::multiply_integers(t.sizes().slice(lead)) * (int64_t)t.element_size();
    from.push_back(pointer(in.back())), to.push_back(pointer(out.back())), bytes.push_back(out.back().numel() ? row : 0);
  }
  if (!in.empty())
    check_rc(abi.reorder_rows((int)in.size(), from.data(), to.data(), bytes.data(), (const int64_t*)pointer(sources), (int)B, (int)K, (int)beam, current_stream(sources.device())));
  return out;
}

void init(const py::dict& symbols) {
  take(abi.last_error, symbols, "rtn_model_ops_last_error");
  take(abi.delta_fwd_workspace_bytes, symbols, "rtn_delta_rule_fwd_workspace_bytes");
  take(abi.delta_saved_bytes, symbols, "rtn_delta_rule_saved_bytes");
  take(abi.delta_fwd, symbols, "rtn_delta_rule_fwd");
  take(abi.delta_bwd_workspace_bytes, symbols, "rtn_delta_rule_bwd_workspace_bytes");
  take(abi.delta_bwd, symbols, "rtn_delta_rule_bwd");
  take(abi.embedding_fwd, symbols, "rtn_embedding_fwd");
  take(abi.embedding_bwd_workspace_bytes, symbols, "rtn_embedding_bwd_workspace_bytes");
  take(abi.embedding_bwd, symbols, "rtn_embedding_bwd");
  take(abi.beam_workspace_bytes, symbols, "rtn_beam_select_workspace_bytes");
  take(abi.beam_select, symbols, "rtn_beam_select");
  take(abi.reorder_rows, symbols, "rtn_reorder_rows");
  ready = true;
}

}  // namespace

PYBIND11_MODULE(_rtn_model, m) {
  m.def("init", &init);
  m.def("gated_delta_rule", &gated_delta_rule);
  m.def("embed", &embed);
  m.def("beam_select", &beam_select);
  m.def("reorder_states", &reorder_states);
}
