// The torch binding of the operators around the stack: embedding, layer norm,
// clipping, beam step.  Their calls are short, and what the host does for one is
// most of the time of a small one: from Python through ctypes a lookup of 256 ids
// took 7.6 us, from here 4.8; a beam step with 24 state planes 52 and 23; the layer
// norm of 64 rows forward and backward 55 to 108 and 35 to 64, because autograd runs
// a backward on a thread of its own, where a node in Python costs it the interpreter
// beside the launches.
//
// Every function checks what the kernels assume and returns None for arguments
// that it does not take; the Python callers then say what is wrong with them.  What
// torch would lose track of is refused here: tensors that require grad where there is
// no backward, tangents, tracing, and memory that is shared with what is written.
#include <algorithm>
#include <map>
#include <set>

#include "native.h"

namespace {

// ---------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------
Tensor embedding_forward(const Tensor& tokens, const Tensor& weight, double scale) {
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor y = at::empty(shape, weight.options());
  check(sparc_embedding_forward(tokens.numel(), weight.size(0), weight.size(1), code_of(weight.scalar_type()),
                                static_cast<int32_t>(tokens.element_size()), tokens.data_ptr(), weight.data_ptr(),
                                static_cast<float>(scale), y.data_ptr(), stream_of(weight)),
        "sparc_embedding_forward");
  return y;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& tokens, double scale,
                        int64_t padding_id) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding_id"] = padding_id;
    return embedding_forward(tokens, contiguous(weight), scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (at::GradMode::is_enabled()) throw std::runtime_error("embedding is not twice differentiable");
    const Tensor tokens = ctx->get_saved_variables()[0], dy = contiguous(grads[0]);
    const c10::DeviceGuard guard(dy.device());
    const int64_t n = tokens.numel(), vocab = ctx->saved_data["vocab"].toInt(), dim = dy.size(-1);
    Tensor dw = at::empty({vocab, dim}, dy.options());
    const size_t need = sparc_embedding_workspace_bytes(n, vocab, dim);
    const Tensor ws = scratch(need, dy);
    check(sparc_embedding_backward(n, vocab, dim, code_of(dy.scalar_type()),
                                   static_cast<int32_t>(tokens.element_size()), tokens.data_ptr(),
                                   ctx->saved_data["padding_id"].toInt(), dy.data_ptr(),
                                   static_cast<float>(ctx->saved_data["scale"].toDouble()), dw.data_ptr(),
                                   ws.data_ptr(), need, stream_of(dy)),
          "sparc_embedding_backward");
    return {dw, Tensor(), Tensor(), Tensor()};
  }
};

optional<Tensor> embedding(const Tensor& tokens, const Tensor& weight, double scale, optional<int64_t> padding) {
  refuse_tracing("embedding");
  if (weight.dim() != 2 || weight.numel() == 0 || !is_io(weight) || !beside(weight, weight) ||
      (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt) || !beside(tokens, weight))
    return std::nullopt;
  const int64_t vocab = weight.size(0);
  if (padding && (*padding < -vocab || *padding >= vocab)) return std::nullopt;
  const int64_t padding_id = !padding ? -1 : *padding < 0 ? *padding + vocab : *padding;
  refuse_tangents("embedding", {&weight});
  const c10::DeviceGuard guard(weight.device());
  if (weight.requires_grad() && at::GradMode::is_enabled())
    return Embedding::apply(weight, contiguous(tokens), scale, padding_id);
  return embedding_forward(contiguous(tokens), contiguous(weight), scale);
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
// x, weight and bias contiguous, weight and bias perhaps undefined
Tensor layer_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, float* mean,
                          float* rstd) {
  const Tensor& p = weight.defined() ? weight : bias.defined() ? bias : x;
  const int64_t cols = x.size(-1);
  Tensor y = at::empty_like(x);
  check(sparc_layer_norm_forward(x.numel() / cols, cols, code_of(x.scalar_type()), code_of(p.scalar_type()),
                                 x.data_ptr(), address(weight), address(bias), static_cast<float>(eps), y.data_ptr(),
                                 mean, rstd, stream_of(x)),
        "sparc_layer_norm_forward");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const optional<Tensor>& weight_in,
                        const optional<Tensor>& bias_in, double eps) {
    const Tensor x = contiguous(x_in), weight = contiguous(weight_in), bias = contiguous(bias_in);
    const int64_t rows = x.numel() / x.size(-1);
    Tensor stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    float* mean = stats.data_ptr<float>();
    const Tensor& p = weight.defined() ? weight : bias.defined() ? bias : x;
    ctx->save_for_backward({x, weight, stats});
    ctx->saved_data["parameters"] = static_cast<int64_t>(p.scalar_type());
    ctx->saved_data["bias"] = bias.defined();
    return layer_norm_forward(x, weight, bias, eps, mean, mean + rows);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (at::GradMode::is_enabled()) throw std::runtime_error("layer_norm is not twice differentiable");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &stats = saved[2];
    const Tensor dy = contiguous(grads[0]);
    const c10::DeviceGuard guard(x.device());
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["parameters"].toInt());
    const auto gradient = [&](bool wanted) { return wanted ? at::empty({cols}, x.options().dtype(type)) : Tensor(); };
    // the inputs are numbered without those that are not there
    Tensor dx = ctx->needs_input_grad(0) ? at::empty_like(x) : Tensor();
    Tensor dw = gradient(weight.defined() && ctx->needs_input_grad(1));
    Tensor db = gradient(ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(weight.defined() ? 2 : 1));
    const size_t need = dw.defined() || db.defined() ? sparc_layer_norm_workspace_bytes(rows, cols) : 0;
    const Tensor ws = need ? scratch(need, x) : Tensor();
    const float* mean = stats.data_ptr<float>();
    check(sparc_layer_norm_backward(rows, cols, code_of(x.scalar_type()), code_of(type), x.data_ptr(), address(weight),
                                    mean, mean + rows, dy.data_ptr(), address(dx), address(dw), address(db),
                                    address(ws), need, stream_of(x)),
          "sparc_layer_norm_backward");
    return {dx, dw, db, Tensor()};
  }
};

optional<Tensor> layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  refuse_tracing("layer_norm");
  if (x.dim() < 1 || x.size(-1) < 1 || !(eps >= 0.0) || !is_io(x) || !beside(x, x)) return std::nullopt;
  for (const auto* p : {&weight, &bias}) {
    if (*p && ((*p)->dim() != 1 || (*p)->numel() != x.size(-1) ||
               ((*p)->scalar_type() != x.scalar_type() && (*p)->scalar_type() != at::kFloat) || !beside(**p, x)))
      return std::nullopt;
  }
  if (weight && bias && weight->scalar_type() != bias->scalar_type()) return std::nullopt;
  refuse_tangents("layer_norm", {&x, pointer(weight), pointer(bias)});
  const c10::DeviceGuard guard(x.device());
  const auto wants = [](const optional<Tensor>& t) { return t && t->requires_grad(); };
  if ((x.requires_grad() || wants(weight) || wants(bias)) && at::GradMode::is_enabled())
    return LayerNorm::apply(x, weight, bias, eps);
  return layer_norm_forward(contiguous(x), contiguous(weight), contiguous(bias), eps, nullptr, nullptr);
}

// ---------------------------------------------------------------------------
// the gradients' norm
// ---------------------------------------------------------------------------
// A tensor's values from its first one on: every sum of i step with i up to most
struct Term { int64_t step, most; };
// Whether such a sum over the terms from the k-th on is ``rest``; steps falling,
// reach[k]: the largest sum from there on.  Strides that nest leave two or three
// values of i to try; after ``tries`` it is taken to be.
bool reaches(const std::vector<Term>& terms, const std::vector<int64_t>& reach, size_t k, int64_t rest, int& tries) {
  if (k == terms.size() || --tries < 0) return true;
  const Term& t = terms[k];
  const int64_t behind = rest - reach[k + 1], least = behind > 0 ? (behind + t.step - 1) / t.step : 0;
  for (int64_t i = std::min(t.most, rest / t.step); i >= least; --i)
    if (reaches(terms, reach, k + 1, rest - i * t.step, tries)) return true;
  return false;
}
// Whether a and b, which starts no sooner, share a byte.  With i and j counting in a
// and b, and j from its end: a value of a lies where one of b does if sum i step + sum
// j step = b - a + the length of b.
bool share_memory(const Tensor& a, const Tensor& b) {
  std::map<int64_t, int64_t, std::greater<>> most;
  int64_t rest = static_cast<char*>(b.data_ptr()) - static_cast<char*>(a.data_ptr());
  const auto add = [&](const Tensor& t, int64_t of_length) {
    const auto dimension = [&](int64_t step, int64_t n) {
      if (n > 1 && step > 0) most[step] += n - 1;
      rest += of_length * (n - 1) * step;
    };
    const int64_t size_of = static_cast<int64_t>(t.element_size());
    for (int64_t d = 0; d < t.dim(); ++d) dimension(t.stride(d) * size_of, t.size(d));
    dimension(1, size_of);
  };
  add(a, 0);
  add(b, 1);
  std::vector<Term> terms;
  for (const auto& [step, n] : most) terms.push_back({step, n});
  std::vector<int64_t> reach(terms.size() + 1, 0);
  for (size_t k = terms.size(); k-- > 0;) reach[k] = reach[k + 1] + terms[k].step * terms[k].most;
  int tries = 1 << 14;
  return rest <= reach[0] && reaches(terms, reach, 0, rest, tries);
}
// Tensors with gaps must not share values: each is scaled in a copy of its own.
void check_apart(Tensors tensors) {
  std::sort(tensors.begin(), tensors.end(), [](const Tensor& a, const Tensor& b) { return a.data_ptr() < b.data_ptr(); });
  for (size_t i = 0; i < tensors.size(); ++i) {
    const auto end = static_cast<char*>(tensors[i].data_ptr()) + reach_of(tensors[i]);
    for (size_t j = i + 1; j < tensors.size() && tensors[j].data_ptr() < end; ++j)
      if (share_memory(tensors[i], tensors[j])) throw std::runtime_error("gradient clipping: two tensors overlap");
  }
}

// A tensor given twice counts once.  max_norm: scale to it.  copies: also tensors with
// gaps between their values and views that negate, by way of a copy.
optional<Tensor> grad_norm(const Tensors& tensors, optional<double> max_norm, bool copies) {
  const char* const what = max_norm ? "clip_grad_norm_" : "grad_norm";
  refuse_tracing(what);
  if (tensors.empty()) return std::nullopt;
  const auto in_place = [](const Tensor& t) { return t.is_non_overlapping_and_dense() && is_literal(t); };
  for (const Tensor& t : tensors)
    if (!beside(t, tensors[0]) || !is_io(t) || !(copies || in_place(t))) return std::nullopt;
  refuse_tangents(what, tensors);
  if (!max_norm) refuse_gradients(what, tensors);
  const size_t n = tensors.size();
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(tensors[0].device());
  // values in a row in memory, in whatever order, are one array; others have a layout
  using Key = std::tuple<void*, int64_t, int32_t, bool, std::vector<int64_t>>;
  std::vector<void*> data;
  std::vector<int64_t> sizes;
  std::vector<int32_t> types;
  std::vector<std::pair<Tensor, Tensor>> copied;  // and their copies
  Tensors distinct;                               // with values, where there are copies
  std::set<Key> seen;
  bool rising = !copies;  // addresses in order are no repeats: nothing to look up
  for (size_t i = 1; i < n; ++i) rising = rising && tensors[i - 1].data_ptr() < tensors[i].data_ptr();
  for (const Tensor& t : tensors) {
    const bool direct = !copies || in_place(t);
    if (!rising) {
      std::vector<int64_t> layout;
      if (!direct) {
        layout = t.sizes().vec();
        layout.insert(layout.end(), t.strides().begin(), t.strides().end());
      }
      if (!seen.insert(Key(t.data_ptr(), t.numel(), code_of(t.scalar_type()), t.is_neg(), std::move(layout))).second)
        continue;
    }
    if (!direct) copied.emplace_back(t, contiguous(t));
    if (copies && t.numel() > 0) distinct.push_back(t);
    data.push_back((direct ? t : copied.back().second).data_ptr());
    sizes.push_back(t.numel());
    types.push_back(code_of(t.scalar_type()));
  }
  if (max_norm) {
    check_apart(std::move(distinct));
    mark_written(tensors);
  }
  const int64_t count = static_cast<int64_t>(data.size());
  Tensor norm = at::empty({}, tensors[0].options().dtype(at::kFloat));
  const size_t need = sparc_grad_norm_workspace_bytes(count);
  const Tensor ws = scratch(need, tensors[0]);
  float* out = norm.data_ptr<float>();
  if (max_norm) {
    check(sparc_clip_grad_norm(count, data.data(), sizes.data(), types.data(), static_cast<float>(*max_norm), out,
                               ws.data_ptr(), need, stream_of(tensors[0])),
          "sparc_clip_grad_norm");
    for (const auto& [t, copy] : copied) t.copy_(copy);
  } else {
    check(sparc_grad_norm(count, data.data(), sizes.data(), types.data(), out, ws.data_ptr(), need,
                          stream_of(tensors[0])),
          "sparc_grad_norm");
  }
  return norm;
}

// ---------------------------------------------------------------------------
// beam search
// ---------------------------------------------------------------------------
bool is_beams(const Tensor& t, int64_t B, int64_t K, at::ScalarType type, const Tensor& with) {
  return t.dim() == 2 && t.size(0) == B && t.size(1) == K && t.scalar_type() == type && beside(t, with);
}

// (tokens, parents, scores, finished)
optional<std::tuple<Tensor, Tensor, Tensor, optional<Tensor>>> beam_step(const Tensor& logits_in,
                                                                         const Tensor& scores_in,
                                                                         const optional<Tensor>& finished_in,
                                                                         optional<int64_t> eos, int64_t most_beams) {
  refuse_tracing("beam_search_step");
  if (logits_in.dim() != 3 || !is_io(logits_in) || !beside(logits_in, logits_in)) return std::nullopt;
  const int64_t B = logits_in.size(0), K = logits_in.size(1), V = logits_in.size(2);
  if (K < 1 || K > most_beams || V < 1 || !is_beams(scores_in, B, K, at::kFloat, logits_in) ||
      (finished_in && (!eos || !is_beams(*finished_in, B, K, at::kBool, logits_in))) ||
      (eos && (*eos < 0 || *eos >= V)))
    return std::nullopt;
  refuse_tangents("beam_search_step", {&logits_in, &scores_in});
  refuse_gradients("beam_search_step", {&logits_in, &scores_in});
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(logits_in.device());
  Tensor logits = logits_in;
  int64_t stride = K > 1 ? logits.stride(1) : B > 1 ? logits.stride(0) : V;
  if (!is_literal(logits) || (V > 1 && logits.stride(2) != 1) || stride < V ||
      (B > 1 && logits.stride(0) != K * stride)) {
    logits = contiguous(logits);
    stride = V;
  }
  const Tensor scores = contiguous(scores_in), finished = contiguous(finished_in);
  const auto make = [&](at::ScalarType type) { return at::empty({B, K}, scores.options().dtype(type)); };
  Tensor tokens = make(at::kLong), parents = make(at::kLong), new_scores = make(at::kFloat);
  optional<Tensor> new_finished;
  if (eos) new_finished = make(at::kBool);
  const size_t need = sparc_beam_workspace_bytes(B, K, V);
  const Tensor ws = scratch(need, scores);
  check(sparc_beam_step(B, K, V, stride, code_of(logits.scalar_type()), logits.data_ptr(), scores.data_ptr<float>(),
                        static_cast<const uint8_t*>(address(finished)), eos ? *eos : -1, tokens.data_ptr<int64_t>(),
                        parents.data_ptr<int64_t>(), new_scores.data_ptr<float>(),
                        eos ? static_cast<uint8_t*>(new_finished->data_ptr()) : nullptr, ws.data_ptr(), need,
                        stream_of(logits)),
        "sparc_beam_step");
  return std::make_tuple(tokens, parents, new_scores, new_finished);
}

// n contiguous tensors like the contiguous ``like``, in one allocation.  (unbind
// makes them by way of the dispatcher: 24 of them 7.5 us, here 3.)
Tensors fresh(size_t n, const Tensor& like) {
  std::vector<int64_t> shape = like.sizes().vec();
  shape.insert(shape.begin(), static_cast<int64_t>(n));
  const Tensor all = at::empty(shape, like.options());
  Tensors parts;
  for (size_t i = 0; i < n; ++i) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(static_cast<int64_t>(i) * like.numel());
    t.unsafeGetTensorImpl()->set_sizes_contiguous(like.sizes());
    parts.push_back(std::move(t));
  }
  return parts;
}

// Whether the tensors of ``out`` overlap neither one another nor a plane that they
// do not replace
bool apart(const Tensors& planes, const Tensors& out) {
  std::vector<std::tuple<uintptr_t, uintptr_t, bool>> spans;  // first byte, end, whether it is written
  for (size_t i = 0; i < out.size(); ++i) {
    const auto at = reinterpret_cast<uintptr_t>(out[i].data_ptr());
    const auto src = reinterpret_cast<uintptr_t>(planes[i].data_ptr());
    if (out[i].numel() == 0) continue;
    spans.emplace_back(at, at + out[i].nbytes(), true);
    if (src == at) continue;
    spans.emplace_back(src, src + reach_of(planes[i]), false);
  }
  std::sort(spans.begin(), spans.end());
  uintptr_t end = 0, written_end = 0;
  for (const auto& [first, last, written] : spans) {
    if (first < (written ? end : written_end)) return false;
    end = std::max(end, last);
    if (written) written_end = std::max(written_end, last);
  }
  return true;
}

// The planes in the parents' order: in ``out`` (of the planes' shapes and types,
// contiguous), or in fresh tensors, which share an allocation where all planes are
// alike.
optional<Tensors> reorder(const Tensors& planes, const Tensor& parents_in, const optional<Tensors>& out) {
  refuse_tracing("reorder_states");
  if (parents_in.dim() != 2 || parents_in.scalar_type() != at::kLong || !beside(parents_in, parents_in))
    return std::nullopt;
  const int64_t B = parents_in.size(0), K = parents_in.size(1), rows = B * K;
  bool alike = true;
  for (const Tensor& p : planes) {
    if (!beside(p, parents_in) || p.dim() < 1 || p.size(0) != rows) return std::nullopt;
    if (rows > 0 && p.numel() / rows * static_cast<int64_t>(p.element_size()) % 2) return std::nullopt;
    alike = alike && p.scalar_type() == planes[0].scalar_type() && p.sizes() == planes[0].sizes();
  }
  if (planes.empty()) return Tensors();
  refuse_tangents("reorder_states", planes);
  refuse_gradients("reorder_states", planes);
  if (out) {
    refuse_tangents("reorder_states", *out);
    refuse_gradients("reorder_states", *out);
  }
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(parents_in.device());
  const Tensor parents = contiguous(parents_in);
  Tensors to;
  if (out) {
    to = *out;
    if (to.size() != planes.size()) return std::nullopt;
    for (size_t i = 0; i < to.size(); ++i)
      if (!beside(to[i], parents) || to[i].scalar_type() != planes[i].scalar_type() ||
          to[i].sizes() != planes[i].sizes() || !to[i].is_contiguous() || !is_literal(to[i]))
        return std::nullopt;
    if (!apart(planes, to))
      throw pybind11::value_error("a tensor of out_states overlaps another one, or another one of the states");
    mark_written(to);
  } else if (alike) {
    to = fresh(planes.size(), planes[0]);
  } else {
    for (const Tensor& p : planes) to.push_back(at::empty(p.sizes(), p.options()));
  }
  Tensors from;  // kept until the launch is enqueued
  std::vector<const void*> src;
  std::vector<void*> dst;
  std::vector<int64_t> bytes;
  for (size_t i = 0; i < planes.size(); ++i) {
    from.push_back(contiguous(planes[i]));
    src.push_back(from[i].data_ptr());
    dst.push_back(to[i].data_ptr());
    bytes.push_back(rows > 0 ? planes[i].numel() / rows * static_cast<int64_t>(planes[i].element_size()) : 0);
  }
  check(sparc_reorder_states(B, K, static_cast<int64_t>(planes.size()), src.data(), dst.data(), bytes.data(),
                             parents.data_ptr<int64_t>(), stream_of(parents)),
        "sparc_reorder_states");
  return to;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("embedding", &embedding);
  m.def("layer_norm", &layer_norm);
  m.def("grad_norm", &grad_norm);
  m.def("beam_step", &beam_step);
  m.def("reorder", &reorder);
  bind_block(m);
}
