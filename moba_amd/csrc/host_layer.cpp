// The host's side of the operators around the attention, for the extension module of host.cpp: what moba_amd/norm_rope.py
// and moba_amd/paged.py ask of their tensors, the allocations, and the calls into libmoba_hip.so.
//
// For one token a step's operators are 4 to 14 us of work for the device each, and were 21 to 23 us for the host in Python; the
// norm's forward and backward of a training step, 76 us on the device, were 186 us in a call through a Python autograd function.
//
// Every function takes the ordinary call -- tensors of the right kind that are read where they lie -- and answers
// NotImplemented to any other, which the caller's own path then checks, copies or refuses.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "host_layer.h"
#include "host_tensors.h"

namespace {

decltype(&moba_qk_norm_rope) norm_call = nullptr;
decltype(&moba_qk_norm_rope_bwd) norm_bwd_call = nullptr;
decltype(&moba_qk_norm_rope_bwd_workspace_bytes) norm_bwd_bytes = nullptr;
decltype(&moba_paged_append) append_call = nullptr;
decltype(&moba_paged_attention) attention_call = nullptr;
decltype(&moba_paged_attention_workspace_bytes) attention_bytes = nullptr;

constexpr int64_t kMostNormTokens = 1 << 25, kMostHeadDim = 128;

// A leaf's gradient arrives on the stream that its node was made on.  A node that an eager graph keeps alive has another stream than
// a capture, whose backward pass would have that stream wait for the captured one, and end the process: refused beforehand.
void check_leaves(std::initializer_list<const Tensor*> leaves, const at::Device& device) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const c10::hip::HIPStream captured = c10::hip::getCurrentHIPStream(device.index());
  for (const Tensor* t : leaves) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!stream || (stream->id() == captured.id() && stream->device_index() == captured.device_index()),
                "qk_norm_rope: an eager graph with the same leaves is alive, whose gradients belong to another stream than "
                "the one being captured: let go of its outputs first");
  }
}

// ---- qk_norm_rope
struct NormArgs {
  Tensor q, k, positions, inv_freq, q_weight, k_weight;
  double eps;
  bool interleaved;
};

bool weight_fits(const Tensor& w, const NormArgs& a) {
  return !w.defined() || ((w.scalar_type() == a.q.scalar_type() || w.scalar_type() == at::kFloat) && w.dim() == 1 && w.is_contiguous() &&
                          w.size(0) == a.q.size(2) && w.device() == a.q.device() && aligned(w, 8));
}
bool norm_fits(const NormArgs& a, int64_t* strides) {
  const Tensor &q = a.q, &k = a.k;
  if (!q.is_cuda() || k.device() != q.device() || !half_type(q) || k.scalar_type() != q.scalar_type() || q.dim() != 3 || k.dim() != 3)
    return false;
  const auto qs = q.sizes(), ks = k.sizes();
  if (qs[0] != ks[0] || qs[2] != ks[2] || qs[0] < 1 || qs[0] > kMostNormTokens || qs[1] < 1 || ks[1] < 1 || qs[1] > kMostHeads ||
      ks[1] > kMostHeads || qs[2] < 8 || qs[2] > kMostHeadDim || qs[2] % 8)
    return false;
  if ((a.positions.scalar_type() != at::kInt && a.positions.scalar_type() != at::kLong) || a.positions.dim() != 1 ||
      !a.positions.is_contiguous() || a.positions.size(0) != qs[0] || a.positions.device() != q.device())
    return false;
  if (!frequencies_fit(a.inv_freq, q.device(), qs[2]) || !weight_fits(a.q_weight, a) || !weight_fits(a.k_weight, a)) return false;
  if (a.q_weight.defined() && a.k_weight.defined() && a.q_weight.scalar_type() != a.k_weight.scalar_type()) return false;
  return a.eps >= 0 && rows_in_place(q, 4, 8, strides) && rows_in_place(k, 4, 8, strides + 2);
}
bool weights_f32(const NormArgs& a) {
  return (a.q_weight.defined() && a.q_weight.scalar_type() == at::kFloat) || (a.k_weight.defined() && a.k_weight.scalar_type() == at::kFloat);
}
std::pair<Tensor, Tensor> norm_forward(const NormArgs& a, const int64_t* strides) {
  const c10::OptionalDeviceGuard guard(a.q.device());
  Tensor yq = fresh_like(a.q), yk = fresh_like(a.k);
  check(norm_call(pointer(a.q), pointer(a.k), mutable_pointer(yq), mutable_pointer(yk), pointer(a.q_weight), pointer(a.k_weight),
                  pointer(a.positions), (const float*)pointer(a.inv_freq), a.q.size(0), (int)a.q.size(1), (int)a.k.size(1),
                  (int)a.q.size(2), (int)(2 * a.inv_freq.numel()), strides, a.positions.scalar_type() == at::kLong ? 64 : 32,
                  a.interleaved, weights_f32(a), (float)a.eps, type_code(a.q), stream_of(a.q)),
        "moba_qk_norm_rope");
  return {yq, yk};
}

struct NormRope : torch::autograd::Function<NormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k,
                                                const Tensor& positions, const Tensor& inv_freq,
                                                const std::optional<Tensor>& q_weight, const std::optional<Tensor>& k_weight,
                                                double eps, bool interleaved) {
    const NormArgs a = {q, k, positions, inv_freq, q_weight.value_or(Tensor()), k_weight.value_or(Tensor()), eps, interleaved};
    int64_t strides[4];
    TORCH_CHECK(norm_fits(a, strides), "qk_norm_rope: tensors that changed on the way");
    ctx->save_for_backward({q, k, positions, inv_freq, a.q_weight, a.k_weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    auto y = norm_forward(a, strides);
    return {y.first, y.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    NormArgs a = {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], ctx->saved_data["eps"].toDouble(),
                  ctx->saved_data["interleaved"].toBool()};
    torch::autograd::variable_list grads(8);
    TORCH_CHECK(!has_tangent(dy[0]) && !has_tangent(dy[1]),
                "qk_norm_rope has no forward-mode derivatives: tensors with a tangent are refused");
    {
      const at::NoGradGuard no_grad;
      const c10::OptionalDeviceGuard guard(a.q.device());
      auto packed = [](const Tensor& g) {
        Tensor t = g.contiguous();
        return aligned(t, 16) ? t : t.clone();
      };
      int64_t strides[4];
      if (!norm_fits(a, strides)) {   // (hooks on saved tensors may give back copies that lie otherwise)
        for (Tensor* t : {&a.q, &a.k, &a.positions, &a.inv_freq, &a.q_weight, &a.k_weight})
          if (t->defined()) *t = packed(*t);
        TORCH_CHECK(norm_fits(a, strides), "qk_norm_rope: saved tensors that changed");
      }
      const Tensor dyq = packed(dy[0]), dyk = packed(dy[1]);
      Tensor dq = fresh_like(a.q), dk = fresh_like(a.k), dqw, dkw, space;
      // (the graph's edges are numbered by the tensors there are: a side without a weight has none)
      if (a.q_weight.defined() && ctx->needs_input_grad(4)) dqw = fresh_like(a.q_weight);
      if (a.k_weight.defined() && ctx->needs_input_grad(a.q_weight.defined() ? 5 : 4)) dkw = fresh_like(a.k_weight);
      if (dqw.defined() || dkw.defined())
        space = bytes(norm_bwd_bytes(a.q.size(0), (int)a.q.size(2)), a.q.device());
      check(norm_bwd_call(pointer(dyq), pointer(dyk), pointer(a.q), pointer(a.k), mutable_pointer(dq), mutable_pointer(dk),
                          pointer(a.q_weight), pointer(a.k_weight), mutable_pointer(dqw), mutable_pointer(dkw),
                          mutable_pointer(space), pointer(a.positions), (const float*)pointer(a.inv_freq), a.q.size(0),
                          (int)a.q.size(1), (int)a.k.size(1), (int)a.q.size(2), (int)(2 * a.inv_freq.numel()), strides,
                          a.positions.scalar_type() == at::kLong ? 64 : 32, a.interleaved, weights_f32(a), (float)a.eps,
                          type_code(a.q), stream_of(a.q)),
            "moba_qk_norm_rope_bwd");
      grads[0] = dq;
      grads[1] = dk;
      grads[4] = dqw;
      grads[5] = dkw;
    }
    // the gradients are not differentiable themselves: asked for with create_graph, they say so when they are differentiated
    if (at::GradMode::is_enabled()) {
      torch::autograd::variable_list defined;
      for (const Tensor& g : grads)
        if (g.defined()) defined.push_back(g);
      const auto error = std::make_shared<torch::autograd::DelayedError>("qk_norm_rope is differentiable once", (int64_t)defined.size());
      defined = (*error)(std::move(defined));
      size_t at = 0;
      for (Tensor& g : grads)
        if (g.defined()) g = defined[at++];
    }
    return grads;
  }
};

}  // namespace

// check_leaves(q, k, q_weight, k_weight), for the caller's own path
PyObject* py_check_leaves(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 4 && THPVariable_Check(args[0]), "check_leaves takes four tensors");
  Tensor t[4];
  for (int i = 0; i < 4; ++i)
    if (THPVariable_Check(args[i])) t[i] = THPVariable_Unpack(args[i]);
  check_leaves({&t[0], &t[1], &t[2], &t[3]}, t[0].device());
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, interleaved)
PyObject* py_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8 && norm_call, "norm_rope takes eight arguments, and the library's entry points");
  const Tensor *q = plain_tensor(args[0]), *k = plain_tensor(args[1]), *at = plain_tensor(args[2]), *f = plain_tensor(args[3]);
  NormArgs a;
  if (!q || !k || !at || !f || !optional_tensor(args[4], a.q_weight) || !optional_tensor(args[5], a.k_weight)) Py_RETURN_NOTIMPLEMENTED;
  a.q = *q; a.k = *k; a.positions = *at; a.inv_freq = *f;
  a.eps = PyFloat_AsDouble(args[6]);
  if (PyErr_Occurred()) return nullptr;
  const int interleaved = PyObject_IsTrue(args[7]);
  if (interleaved < 0) return nullptr;
  a.interleaved = interleaved;
  for (const Tensor* t : {&a.q, &a.k, &a.inv_freq, &a.q_weight, &a.k_weight})
    if (has_tangent(*t)) Py_RETURN_NOTIMPLEMENTED;
  if (a.inv_freq.requires_grad() && at::GradMode::is_enabled()) Py_RETURN_NOTIMPLEMENTED;
  int64_t strides[4];
  if (!norm_fits(a, strides)) Py_RETURN_NOTIMPLEMENTED;
  auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
  std::pair<Tensor, Tensor> y;
  {
    const NoGil no_gil;
    if (at::GradMode::is_enabled() && (wants(a.q) || wants(a.k) || wants(a.q_weight) || wants(a.k_weight))) {
      check_leaves({&a.q, &a.k, &a.q_weight, &a.k_weight}, a.q.device());
      auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      const auto out =
          NormRope::apply(a.q, a.k, a.positions, a.inv_freq, given(a.q_weight), given(a.k_weight), a.eps, a.interleaved);
      y = {out[0], out[1]};
    } else {
      y = norm_forward(a, strides);
    }
  }
  PyObject *const first = THPVariable_Wrap(y.first), *const second = first ? THPVariable_Wrap(y.second) : nullptr;
  if (!second) {
    Py_XDECREF(first);
    return nullptr;
  }
  PyObject* const pair = PyTuple_New(2);
  if (!pair) {
    Py_DECREF(first);
    Py_DECREF(second);
    return nullptr;
  }
  PyTuple_SET_ITEM(pair, 0, first);
  PyTuple_SET_ITEM(pair, 1, second);
  return pair;
  END_HANDLE_TH_ERRORS
}

// paged_append(k_pages, v_pages, k_scales, v_scales, key, value, page_table, lengths, cu_new, inv_freq, query, interleaved)
PyObject* py_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 12 && append_call, "paged_append takes twelve arguments, and the library's entry points");
  Cache cache;
  Index index;
  const Tensor *key = plain_tensor(args[4]), *value = plain_tensor(args[5]);
  Tensor inv_freq, query;
  if (!cache.take(args) || !key || !value || !index.take(args + 6, cache.k->device()) || !optional_tensor(args[9], inv_freq) ||
      !optional_tensor(args[10], query))
    Py_RETURN_NOTIMPLEMENTED;
  const int64_t hkv = cache.k->size(1), d = cache.k->size(3);
  if (!cache.takes_rows(*key) || !cache.takes_rows(*value) || key->sizes() != value->sizes() || key->scalar_type() != value->scalar_type() ||
      key->size(1) != hkv || key->size(0) < 1 || key->size(0) >= (1 << 30))
    Py_RETURN_NOTIMPLEMENTED;
  int64_t strides[7] = {0, 0};
  if (query.defined() && (!cache.takes_rows(query) || query.scalar_type() != key->scalar_type() || query.size(0) != key->size(0) ||
                          query.size(1) < 1 || query.size(1) > kMostHeads || !rows_in_place(query, 4, 8, strides)))
    Py_RETURN_NOTIMPLEMENTED;
  if (wants_derivative(inv_freq)) Py_RETURN_NOTIMPLEMENTED;
  if (inv_freq.defined() && !frequencies_fit(inv_freq, key->device(), d)) Py_RETURN_NOTIMPLEMENTED;
  if (!rows_in_place(*key, 4, 8, strides + 2) || !rows_in_place(*value, 4, 8, strides + 4)) Py_RETURN_NOTIMPLEMENTED;
  strides[6] = index.table->stride(0);
  const int interleaved = PyObject_IsTrue(args[11]);
  if (interleaved < 0) return nullptr;
  Tensor out;
  {
    const Tensor k = *key, v = *value, kp = *cache.k, vp = *cache.v, table = *index.table, lengths = *index.lengths, cu = *index.cu;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(k.device());
    if (query.defined()) out = fresh_like(query);
    check(append_call(pointer(k), pointer(v), pointer(query), mutable_pointer(out), kp.mutable_data_ptr(), vp.mutable_data_ptr(),
                      (float*)mutable_pointer(cache.k_scales), (float*)mutable_pointer(cache.v_scales), (const int32_t*)pointer(table),
                      (const int32_t*)pointer(lengths), (const int32_t*)pointer(cu), (const float*)pointer(inv_freq), k.size(0),
                      (int)table.size(0), query.defined() ? (int)query.size(1) : 0, (int)hkv, (int)d,
                      inv_freq.defined() ? (int)(2 * inv_freq.numel()) : 0, (int)kp.size(2), kp.size(0), table.size(1), strides,
                      cache.k_scales.defined(), interleaved, type_code(k), stream_of(k)),
          "moba_paged_append");
    for (const Tensor& t : {kp, vp, cache.k_scales, cache.v_scales}) written(t);
  }
  if (!out.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_attention(k_pages, v_pages, k_scales, v_scales, query, page_table, lengths, cu_new, scaling, max_new)
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10 && attention_call, "paged_attention takes ten arguments, and the library's entry points");
  Cache cache;
  Index index;
  const Tensor* query = plain_tensor(args[4]);
  if (!cache.take(args) || !query || !index.take(args + 5, cache.k->device()) || !cache.takes_rows(*query)) Py_RETURN_NOTIMPLEMENTED;
  const int64_t tokens = query->size(0), heads = query->size(1), hkv = cache.k->size(1), d = cache.k->size(3);
  int64_t strides[3];
  if (tokens < 1 || tokens >= (1 << 24) || heads < 1 || heads % hkv || tokens * heads > INT32_MAX || !rows_in_place(*query, 8, 16, strides))
    Py_RETURN_NOTIMPLEMENTED;
  strides[2] = index.table->stride(0);
  double scale = d == 128 ? 0.08838834764831845 : 0.125;  // d ** -0.5
  if (args[8] != Py_None) {
    scale = PyFloat_AsDouble(args[8]);
    if (PyErr_Occurred()) return nullptr;
  }
  int64_t max_new = -1;
  if (args[9] != Py_None) {
    max_new = PyLong_AsLongLong(args[9]);
    if (PyErr_Occurred()) return nullptr;
    if (max_new < 0) Py_RETURN_NOTIMPLEMENTED;
    max_new = std::min(max_new, tokens);
  }
  Tensor out;
  {
    const Tensor q = *query, kp = *cache.k, vp = *cache.v, table = *index.table, lengths = *index.lengths, cu = *index.cu;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(q.device());
    out = fresh_like(q);
    const int b = (int)table.size(0);
    Tensor space = bytes(attention_bytes(tokens, b, (int)heads, (int)hkv, (int)d, cache.k_scales.defined(), (int)max_new), q.device());
    check(attention_call(pointer(q), mutable_pointer(out), pointer(kp), pointer(vp), (const float*)pointer(cache.k_scales),
                         (const float*)pointer(cache.v_scales), (const int32_t*)pointer(table), (const int32_t*)pointer(lengths),
                         (const int32_t*)pointer(cu), mutable_pointer(space), tokens, b, (int)heads, (int)hkv, (int)d, (int)kp.size(2),
                         kp.size(0), table.size(1), (int)max_new, strides, cache.k_scales.defined(), (float)scale, type_code(q),
                         stream_of(q)),
          "moba_paged_attention");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind_layer(addresses of moba_qk_norm_rope, moba_qk_norm_rope_bwd, moba_qk_norm_rope_bwd_workspace_bytes, moba_paged_append,
// moba_paged_attention, moba_paged_attention_workspace_bytes, moba_strerror), of the library whose version bind() has checked
PyObject* py_bind_layer(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7, "bind_layer takes seven addresses");
  void* at[7];
  for (int i = 0; i < 7; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  norm_call = reinterpret_cast<decltype(norm_call)>(at[0]);
  norm_bwd_call = reinterpret_cast<decltype(norm_bwd_call)>(at[1]);
  norm_bwd_bytes = reinterpret_cast<decltype(norm_bwd_bytes)>(at[2]);
  append_call = reinterpret_cast<decltype(append_call)>(at[3]);
  attention_call = reinterpret_cast<decltype(attention_call)>(at[4]);
  attention_bytes = reinterpret_cast<decltype(attention_bytes)>(at[5]);
  str_error = reinterpret_cast<decltype(str_error)>(at[6]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
