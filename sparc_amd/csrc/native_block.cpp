// The torch binding of the operators of a linear attention block: norms and rotation
// of queries and keys, linear attention with its step, the gated linear unit.  As in
// native.cpp every function returns None for arguments that it does not take.
#include "native.h"

namespace {

// ---------------------------------------------------------------------------
// common
// ---------------------------------------------------------------------------
// Values of the last dimension in a row, the others at any strides
Tensor rows_of(const Tensor& t) {
  return is_literal(t) && (t.stride(-1) == 1 || t.size(-1) <= 1) ? t : contiguous(t);
}
// The same for sequences [B, T, H, D], where the rows of one head lie apart and not too far
Tensor steps_of(const Tensor& t) {
  const bool fits = t.size(1) <= 1 || (t.stride(1) >= t.size(3) && t.stride(1) < (1 << 22));
  return fits ? rows_of(t) : t.clone(at::MemoryFormat::Contiguous);
}
void strides_of(const Tensor& t, int64_t (&stride)[3]) {  // [B, T, H, D], or one step's [B, H, D]
  const bool one = t.dim() == 3;
  stride[0] = t.stride(0);
  stride[1] = one ? 0 : t.stride(1);
  stride[2] = t.stride(one ? 1 : 2);
}
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const optional<Tensor>& t) { return t && t->requires_grad(); }
// ``t`` as int64, contiguous; undefined where there is none
Tensor as_long(const optional<Tensor>& t) { return t ? t->to(at::kLong).contiguous() : Tensor(); }
bool is_index(const Tensor& t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }
void refuse_twice(const char* what) {
  if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(what) + " is not twice differentiable");
}

// ---------------------------------------------------------------------------
// norms and rotation of queries and keys
// ---------------------------------------------------------------------------
struct RotaryCall {
  Tensor q, k, qw, kw, table, positions;  // qw, kw, positions perhaps undefined
  sparc_rotary_desc desc;
};
RotaryCall rotary_call(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& table,
                       const Tensor& positions, bool interleaved, double eps) {
  RotaryCall c{q, k, qw, kw, table, positions, {}};
  sparc_rotary_desc& d = c.desc;
  d.batch = q.size(0), d.length = q.size(1), d.q_heads = q.size(2), d.head_dim = q.size(3);
  d.k_heads = k.size(2);
  d.rotary_dim = table.size(1), d.table_rows = table.size(0);
  strides_of(q, d.q_stride);
  strides_of(k, d.k_stride);
  const Tensor& p = qw.defined() ? qw : kw.defined() ? kw : q;
  d.io_dtype = code_of(q.scalar_type());
  d.param_dtype = code_of(p.scalar_type());
  d.interleaved = interleaved;
  d.eps = static_cast<float>(eps);
  return c;
}
std::tuple<Tensor, Tensor> rotary_forward(const RotaryCall& c) {
  Tensor yq = at::empty(c.q.sizes(), c.q.options()), yk = at::empty(c.k.sizes(), c.k.options());
  check(sparc_qk_norm_rotary_forward(&c.desc, c.q.data_ptr(), c.k.data_ptr(), address(c.qw), address(c.kw),
                                     c.table.data_ptr<float>(), static_cast<const int64_t*>(address(c.positions)),
                                     yq.data_ptr(), yk.data_ptr(), stream_of(c.q)),
        "sparc_qk_norm_rotary_forward");
  return {yq, yk};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const optional<Tensor>& qw,
                               const optional<Tensor>& kw, const Tensor& table, const optional<Tensor>& positions,
                               bool interleaved, double eps) {
    const RotaryCall c = rotary_call(rows_of(q), rows_of(k), contiguous(qw), contiguous(kw), table.contiguous(),
                                     contiguous(positions), interleaved, eps);
    ctx->save_for_backward({c.q, c.k, c.qw, c.kw, c.table, c.positions});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["eps"] = eps;
    const auto [yq, yk] = rotary_forward(c);
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_twice("qk_norm_rotary");
    const variable_list s = ctx->get_saved_variables();
    const RotaryCall c = rotary_call(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["interleaved"].toBool(),
                                     ctx->saved_data["eps"].toDouble());
    const c10::DeviceGuard guard(c.q.device());
    const Tensor dyq = contiguous(grads[0]), dyk = contiguous(grads[1]);
    // the inputs are numbered without those that are not there
    const auto like = [](const Tensor& t, bool wanted) { return wanted ? at::empty(t.sizes(), t.options()) : Tensor(); };
    Tensor dq = like(c.q, ctx->needs_input_grad(0)), dk = like(c.k, ctx->needs_input_grad(1));
    Tensor dqw = like(c.qw, c.qw.defined() && ctx->needs_input_grad(2));
    Tensor dkw = like(c.kw, c.kw.defined() && ctx->needs_input_grad(c.qw.defined() ? 3 : 2));
    const size_t need = dqw.defined() || dkw.defined() ? sparc_qk_norm_rotary_workspace_bytes(&c.desc) : 0;
    const Tensor ws = need ? scratch(need, c.q) : Tensor();
    check(sparc_qk_norm_rotary_backward(&c.desc, c.q.data_ptr(), c.k.data_ptr(), address(c.qw), address(c.kw),
                                        c.table.data_ptr<float>(), static_cast<const int64_t*>(address(c.positions)),
                                        dyq.data_ptr(), dyk.data_ptr(), address(dq), address(dk), address(dqw),
                                        address(dkw), address(ws), need, stream_of(c.q)),
          "sparc_qk_norm_rotary_backward");
    return {dq, dk, dqw, dkw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

optional<std::tuple<Tensor, Tensor>> qk_norm_rotary(const Tensor& q, const Tensor& k, const optional<Tensor>& qw,
                                                    const optional<Tensor>& kw, const Tensor& table,
                                                    const optional<Tensor>& positions_in, bool interleaved, double eps) {
  refuse_tracing("qk_norm_rotary");
  if (q.dim() != 4 || k.dim() != 4 || !is_io(q) || k.scalar_type() != q.scalar_type() || !beside(q, q) ||
      !beside(k, q) || q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3) ||
      q.size(2) < 1 || k.size(2) < 1 || q.size(3) < 1 || q.size(3) > 512 || !(eps >= 0.0))
    return std::nullopt;
  if (table.dim() != 2 || table.scalar_type() != at::kFloat || !beside(table, q) || table.size(1) > q.size(3) ||
      table.size(1) % 2)
    return std::nullopt;
  for (const auto* p : {&qw, &kw})
    if (*p && ((*p)->dim() != 1 || (*p)->numel() != q.size(3) ||
               ((*p)->scalar_type() != q.scalar_type() && (*p)->scalar_type() != at::kFloat) || !beside(**p, q)))
      return std::nullopt;
  if (qw && kw && qw->scalar_type() != kw->scalar_type()) return std::nullopt;
  optional<Tensor> positions;
  if (positions_in) {
    const Tensor& p = *positions_in;
    if (!is_index(p) || !beside(p, q) || p.dim() < 1 || p.dim() > 2 ||
        (p.size(-1) != q.size(1) && p.size(-1) != 1) || (p.dim() == 2 && p.size(0) != q.size(0) && p.size(0) != 1))
      return std::nullopt;
  }
  refuse_tangents("qk_norm_rotary", {&q, &k, pointer(qw), pointer(kw), &table});
  refuse_gradients("qk_norm_rotary's table", {&table});
  const c10::DeviceGuard guard(q.device());
  if (positions_in) positions = positions_in->to(at::kLong).expand({q.size(0), q.size(1)}).contiguous();
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(qw) || wants(kw))) {
    const variable_list y = Rotary::apply(q, k, qw, kw, table, positions, interleaved, eps);
    return std::make_tuple(y[0], y[1]);
  }
  return rotary_forward(rotary_call(rows_of(q), rows_of(k), contiguous(qw), contiguous(kw), table.contiguous(),
                                    contiguous(positions), interleaved, eps));
}

// ---------------------------------------------------------------------------
// linear attention
// ---------------------------------------------------------------------------
struct LinearCall {
  Tensor q, k, v, decay, state, lengths;  // state and lengths perhaps undefined
  sparc_linear_desc desc;
};
LinearCall linear_call(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const Tensor& state,
                       const Tensor& lengths, double scale) {
  LinearCall c{q, k, v, decay, state, lengths, {}};
  sparc_linear_desc& d = c.desc;
  d.batch = q.size(0), d.length = q.dim() == 3 ? 1 : q.size(1), d.heads = q.size(-2), d.key_dim = q.size(-1);
  d.kv_heads = k.size(-2), d.value_dim = v.size(-1);
  d.io_dtype = code_of(q.scalar_type());
  d.scale = static_cast<float>(scale);
  strides_of(q, d.q_stride);
  strides_of(k, d.k_stride);
  strides_of(v, d.v_stride);
  return c;
}
const float* floats(const Tensor& t) { return static_cast<const float*>(address(t)); }
std::tuple<Tensor, Tensor> linear_forward(const LinearCall& c) {
  const sparc_linear_desc& d = c.desc;
  Tensor o = at::empty({d.batch, d.length, d.heads, d.value_dim}, c.q.options());
  Tensor after = at::empty({d.batch, d.heads, d.key_dim, d.value_dim}, c.decay.options());
  const size_t need = sparc_linear_attention_workspace_bytes(&d, 0);
  const Tensor ws = need ? scratch(need, c.q) : Tensor();
  check(sparc_linear_attention_forward(&d, c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), floats(c.decay),
                                       static_cast<const int64_t*>(address(c.lengths)), floats(c.state), o.data_ptr(),
                                       after.data_ptr<float>(), address(ws), need, stream_of(c.q)),
        "sparc_linear_attention_forward");
  return {o, after};
}

struct Linear : torch::autograd::Function<Linear> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const optional<Tensor>& state, const Tensor& decay, const optional<Tensor>& lengths,
                               double scale) {
    const LinearCall c = linear_call(steps_of(q), steps_of(k), steps_of(v), contiguous(decay), contiguous(state),
                                     contiguous(lengths), scale);
    ctx->save_for_backward({c.q, c.k, c.v, c.decay, c.state, c.lengths});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);  // mostly there is none for the state
    const auto [o, after] = linear_forward(c);
    return {o, after};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_twice("linear_attention");
    const variable_list s = ctx->get_saved_variables();
    const LinearCall c = linear_call(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["scale"].toDouble());
    const c10::DeviceGuard guard(c.q.device());
    const sparc_linear_desc& d = c.desc;
    const Tensor dy = grads[0].defined() ? contiguous(grads[0])
                                         : at::zeros({d.batch, d.length, d.heads, d.value_dim}, c.q.options());
    const Tensor dafter = grads[1].defined() ? contiguous(grads[1]) : Tensor();
    Tensor dq = at::empty(c.q.sizes(), c.q.options()), dk = at::empty(c.k.sizes(), c.q.options());
    Tensor dv = at::empty(c.v.sizes(), c.q.options());
    Tensor dstate;
    if (c.state.defined() && ctx->needs_input_grad(3)) dstate = at::empty(c.state.sizes(), c.state.options());
    const size_t need = sparc_linear_attention_workspace_bytes(&d, 1);
    const Tensor ws = need ? scratch(need, c.q) : Tensor();
    check(sparc_linear_attention_backward(&d, c.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), floats(c.decay),
                                          static_cast<const int64_t*>(address(c.lengths)), floats(c.state),
                                          dy.data_ptr(), floats(dafter), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                          static_cast<float*>(address(dstate)), address(ws), need, stream_of(c.q)),
          "sparc_linear_attention_backward");
    return {dq, dk, dv, dstate, Tensor(), Tensor(), Tensor()};
  }
};

// whether these are what a call over sequences (dim 4) or of one step (dim 3) takes
bool are_linear(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay, const optional<Tensor>& state,
                int64_t dim) {
  if (q.dim() != dim || k.dim() != dim || v.dim() != dim || !is_io(q) || !beside(q, q)) return false;
  for (const Tensor* t : {&k, &v}) {
    if (t->scalar_type() != q.scalar_type() || !beside(*t, q)) return false;
    for (int64_t i = 0; i < dim - 2; ++i)
      if (t->size(i) != q.size(i)) return false;
  }
  const int64_t heads = q.size(-2), kv = k.size(-2);
  const auto fits = [](int64_t n) { return n >= 1 && n <= 256; };
  return heads >= 1 && kv >= 1 && heads % kv == 0 && v.size(-2) == kv && k.size(-1) == q.size(-1) &&
         fits(q.size(-1)) && fits(v.size(-1)) && decay.dim() == 1 && decay.numel() == heads &&
         decay.scalar_type() == at::kFloat && beside(decay, q) &&
         (!state || (state->dim() == 4 && state->scalar_type() == at::kFloat && beside(*state, q) &&
                     state->size(0) == q.size(0) && state->size(1) == heads && state->size(2) == q.size(-1) &&
                     state->size(3) == v.size(-1)));
}

optional<std::tuple<Tensor, Tensor>> linear_attention(const Tensor& q, const Tensor& k, const Tensor& v,
                                                      const Tensor& decay, const optional<Tensor>& state,
                                                      optional<double> scale_in, const optional<Tensor>& lengths_in) {
  refuse_tracing("linear_attention");
  if (!are_linear(q, k, v, decay, state, 4)) return std::nullopt;
  if (lengths_in && (lengths_in->dim() != 1 || lengths_in->numel() != q.size(0) || !is_index(*lengths_in) ||
                     !beside(*lengths_in, q)))
    return std::nullopt;
  refuse_tangents("linear_attention", {&q, &k, &v, &decay, pointer(state)});
  refuse_gradients("linear_attention's decay", {&decay});
  const c10::DeviceGuard guard(q.device());
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q.size(-1)));
  optional<Tensor> lengths;
  if (lengths_in) lengths = as_long(lengths_in);
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(state))) {
    const variable_list y = Linear::apply(q, k, v, state, decay, lengths, scale);
    return std::make_tuple(y[0], y[1]);
  }
  return linear_forward(linear_call(steps_of(q), steps_of(k), steps_of(v), contiguous(decay), contiguous(state),
                                    contiguous(lengths), scale));
}

// Whether the memory that two tensors span overlaps
bool overlap(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto from = [](const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
  return from(a) < from(b) + reach_of(b) && from(b) < from(a) + reach_of(a);
}

optional<std::tuple<Tensor, Tensor>> linear_attention_step(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                                           const Tensor& decay_in, const Tensor& state_in,
                                                           optional<double> scale_in, const optional<Tensor>& out) {
  const char* const what = "linear_attention_step";
  refuse_tracing(what);
  if (!are_linear(q_in, k_in, v_in, decay_in, state_in, 3)) return std::nullopt;
  if (out && (!beside(*out, q_in) || out->scalar_type() != at::kFloat || out->sizes() != state_in.sizes() ||
              !out->is_contiguous() || !is_literal(*out)))
    return std::nullopt;
  refuse_tangents(what, {&q_in, &k_in, &v_in, &decay_in, &state_in, pointer(out)});
  refuse_gradients(what, {&q_in, &k_in, &v_in, &decay_in, &state_in, pointer(out)});
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(q_in.device());
  const Tensor q = rows_of(q_in), k = rows_of(k_in), v = rows_of(v_in);
  const Tensor decay = contiguous(decay_in), state = contiguous(state_in);
  if (out) {
    const bool same = out->data_ptr() == state_in.data_ptr() && state_in.is_contiguous();
    for (const Tensor* t : {&q, &k, &v, &decay})
      if (overlap(*out, *t)) throw pybind11::value_error("out_state overlaps an input");
    if (!same && overlap(*out, state)) throw pybind11::value_error("out_state overlaps the state without being it");
    mark_written({*out});
  }
  Tensor after = out ? *out : at::empty(state.sizes(), state.options());
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q.size(-1)));
  const LinearCall c = linear_call(q, k, v, decay, state, Tensor(), scale);
  Tensor o = at::empty({q.size(0), q.size(1), v.size(2)}, q.options());
  check(sparc_linear_attention_step(&c.desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), floats(decay), floats(state),
                                    o.data_ptr(), after.data_ptr<float>(), stream_of(q)),
        "sparc_linear_attention_step");
  return std::make_tuple(o, after);
}

// ---------------------------------------------------------------------------
// gated linear unit
// ---------------------------------------------------------------------------
// x, wg and wu contiguous
Tensor gated_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  std::vector<int64_t> shape = x.sizes().vec();
  const int64_t dim = shape.back();
  shape.back() = wg.size(0);
  Tensor y = at::empty(shape, x.options());
  check(sparc_gated_forward(x.numel() / dim, dim, wg.size(0), code_of(x.scalar_type()), static_cast<int32_t>(act),
                            x.data_ptr(), wg.data_ptr(), wu.data_ptr(), y.data_ptr(), stream_of(x)),
        "sparc_gated_forward");
  return y;
}

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& wg_in, const Tensor& wu_in,
                        int64_t act) {
    const Tensor x = contiguous(x_in), wg = contiguous(wg_in), wu = contiguous(wu_in);
    ctx->save_for_backward({x, wg, wu});
    ctx->saved_data["act"] = act;
    return gated_forward(x, wg, wu, act);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_twice("gated_linear_unit");
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &wg = s[1], &wu = s[2], dy = contiguous(grads[0]);
    const c10::DeviceGuard guard(x.device());
    const int64_t dim = x.size(-1), hidden = wg.size(0), rows = x.numel() / dim;
    const bool weights = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    Tensor dx = ctx->needs_input_grad(0) ? at::empty_like(x) : Tensor(), dwg, dwu;
    if (weights) dwg = at::empty_like(wg), dwu = at::empty_like(wu);
    const int32_t io = code_of(x.scalar_type());
    const size_t need = sparc_gated_workspace_bytes(rows, dim, hidden, io);
    const Tensor ws = scratch(need, x);
    check(sparc_gated_backward(rows, dim, hidden, io, static_cast<int32_t>(ctx->saved_data["act"].toInt()),
                               x.data_ptr(), wg.data_ptr(), wu.data_ptr(), dy.data_ptr(), address(dx), address(dwg),
                               address(dwu), ws.data_ptr(), need, stream_of(x)),
          "sparc_gated_backward");
    return {dx, ctx->needs_input_grad(1) ? dwg : Tensor(), ctx->needs_input_grad(2) ? dwu : Tensor(), Tensor()};
  }
};

optional<Tensor> gated_linear_unit(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  refuse_tracing("gated_linear_unit");
  if (x.dim() < 1 || x.size(-1) < 1 || !is_io(x) || !beside(x, x)) return std::nullopt;
  for (const Tensor* w : {&wg, &wu})
    if (w->dim() != 2 || w->size(0) < 1 || w->size(1) != x.size(-1) || w->scalar_type() != x.scalar_type() ||
        !beside(*w, x))
      return std::nullopt;
  if (wg.size(0) != wu.size(0)) return std::nullopt;
  refuse_tangents("gated_linear_unit", {&x, &wg, &wu});
  const c10::DeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants(x) || wants(wg) || wants(wu))) return Gated::apply(x, wg, wu, act);
  return gated_forward(contiguous(x), contiguous(wg), contiguous(wu), act);
}

}  // namespace

void bind_block(pybind11::module_& m) {
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("linear_attention", &linear_attention);
  m.def("linear_attention_step", &linear_attention_step);
  m.def("gated_linear_unit", &gated_linear_unit);
}
