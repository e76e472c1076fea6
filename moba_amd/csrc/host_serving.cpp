// The host's side of the operators of serving, for the extension module of host.cpp: moba_amd/paged_prefix.py, paged_blocks.py and
// paged_tables.py, as host_layer.cpp is for the operators around the attention.
//
// Every function takes the ordinary call and answers NotImplemented to any other; the caller then checks, copies, and calls again.
#include "host_layer.h"
#include "host_tensors.h"

namespace {

decltype(&moba_paged_prefix_attention) prefix_call = nullptr;
decltype(&moba_paged_prefix_attention_workspace_bytes) prefix_bytes = nullptr;
decltype(&moba_paged_block_attention) block_call = nullptr;
decltype(&moba_paged_block_attention_workspace_bytes) block_bytes = nullptr;
decltype(&moba_paged_key_sums) sums_call = nullptr;
decltype(&moba_paged_select_blocks) select_call = nullptr;
decltype(&moba_paged_select_blocks_workspace_bytes) select_bytes = nullptr;
decltype(&moba_paged_reserve) reserve_call = nullptr;
decltype(&moba_paged_reserve_workspace_bytes) reserve_bytes = nullptr;
decltype(&moba_paged_release) release_call = nullptr;

constexpr int64_t kMostTokens = 1 << 24;   // fewer than these
constexpr int64_t kMostBlocks = 16384;      // of a row of the table that the selection chooses from

bool ints(const Tensor* t, int64_t dim, const at::Device& device) {
  return t && t->scalar_type() == at::kInt && t->dim() == dim && t->device() == device && t->is_contiguous();
}

// queries of the attention and the selection
bool query_fits(const Tensor& q, int64_t hkv, int64_t* strides) {
  const int64_t tokens = q.size(0), heads = q.size(1);
  return tokens >= 1 && tokens < kMostTokens && heads >= 1 && heads % hkv == 0 && tokens * heads <= INT32_MAX && rows_in_place(q, 8, 16, strides);
}

// a number or None: false with an error set
bool scale_of(PyObject* o, int64_t d, double& scale) {
  scale = d == 128 ? 0.08838834764831845 : 0.125;  // d ** -0.5
  if (o == Py_None) return true;
  scale = PyFloat_AsDouble(o);
  return !PyErr_Occurred();
}

}  // namespace

// paged_prefix_attention(k_pages, v_pages, k_scales, v_scales, query, page_table, lengths, cu_new, cu_groups, shared, scaling)
PyObject* py_paged_prefix_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11 && prefix_call, "paged_prefix_attention takes eleven arguments, and the library's entry points");
  Cache cache;
  Index index;
  const Tensor *query = plain_tensor(args[4]), *groups = plain_tensor(args[8]), *shared = plain_tensor(args[9]);
  if (!cache.take(args) || !query || !index.take(args + 5, cache.k->device()) || !cache.takes_rows(*query)) Py_RETURN_NOTIMPLEMENTED;
  const int64_t hkv = cache.k->size(1), d = cache.k->size(3);
  int64_t strides[3];
  if (!query_fits(*query, hkv, strides) || !ints(groups, 1, cache.k->device()) || !ints(shared, 1, cache.k->device()) ||
      shared->size(0) < 1 || shared->size(0) >= INT32_MAX || groups->size(0) != shared->size(0) + 1)
    Py_RETURN_NOTIMPLEMENTED;
  strides[2] = index.table->stride(0);
  double scale;
  if (!scale_of(args[10], d, scale)) return nullptr;
  Tensor out;
  {
    const Tensor q = *query, kp = *cache.k, vp = *cache.v, table = *index.table, lengths = *index.lengths, cu = *index.cu, cg = *groups,
                 front = *shared;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(q.device());
    out = fresh_like(q);
    const int b = (int)table.size(0), g = (int)front.size(0);
    Tensor space = bytes(prefix_bytes(q.size(0), b, g, (int)q.size(1), (int)hkv, (int)d, cache.k_scales.defined()), q.device());
    check(prefix_call(pointer(q), mutable_pointer(out), pointer(kp), pointer(vp), (const float*)pointer(cache.k_scales),
                      (const float*)pointer(cache.v_scales), (const int32_t*)pointer(table), (const int32_t*)pointer(lengths),
                      (const int32_t*)pointer(cu), (const int32_t*)pointer(cg), (const int32_t*)pointer(front), mutable_pointer(space),
                      q.size(0), b, g, (int)q.size(1), (int)hkv, (int)d, (int)kp.size(2), kp.size(0), table.size(1), strides,
                      cache.k_scales.defined(), (float)scale, type_code(q), stream_of(q)),
          "moba_paged_prefix_attention");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_block_attention(k_pages, v_pages, k_scales, v_scales, query, page_table, lengths, cu_new, blocks, block_size, scaling)
PyObject* py_paged_block_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11 && block_call, "paged_block_attention takes eleven arguments, and the library's entry points");
  Cache cache;
  Index index;
  const Tensor *query = plain_tensor(args[4]), *blocks = plain_tensor(args[8]);
  if (!cache.take(args) || !query || !index.take(args + 5, cache.k->device()) || !cache.takes_rows(*query)) Py_RETURN_NOTIMPLEMENTED;
  const int64_t hkv = cache.k->size(1), d = cache.k->size(3), block_size = PyLong_AsLongLong(args[9]);
  if (PyErr_Occurred()) return nullptr;
  int64_t strides[3];
  if (!query_fits(*query, hkv, strides) || !ints(blocks, 3, cache.k->device()) || blocks->size(0) != query->size(0) ||
      blocks->size(1) != query->size(1) || blocks->size(2) < 1 || blocks->size(2) > 64 || block_size < 1 || block_size > (1 << 24) ||
      block_size % cache.k->size(2))
    Py_RETURN_NOTIMPLEMENTED;
  strides[2] = index.table->stride(0);
  double scale;
  if (!scale_of(args[10], d, scale)) return nullptr;
  Tensor out;
  {
    const Tensor q = *query, kp = *cache.k, vp = *cache.v, table = *index.table, lengths = *index.lengths, cu = *index.cu, picks = *blocks;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(q.device());
    out = fresh_like(q);
    const int b = (int)table.size(0), h = (int)q.size(1), page = (int)kp.size(2), topk = (int)picks.size(2);
    Tensor space = bytes(block_bytes(q.size(0), b, h, (int)hkv, (int)d, page, table.size(1), (int)block_size, topk, cache.k_scales.defined()),
                         q.device());
    check(block_call(pointer(q), mutable_pointer(out), pointer(kp), pointer(vp), (const float*)pointer(cache.k_scales),
                     (const float*)pointer(cache.v_scales), (const int32_t*)pointer(picks), (const int32_t*)pointer(table),
                     (const int32_t*)pointer(lengths), (const int32_t*)pointer(cu), mutable_pointer(space), q.size(0), b, h, (int)hkv,
                     (int)d, page, kp.size(0), table.size(1), (int)block_size, topk, strides, cache.k_scales.defined(), (float)scale,
                     type_code(q), stream_of(q)),
          "moba_paged_block_attention");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_key_sums(k_pages, v_pages, k_scales, v_scales, sums, page_table, lengths, cu_new, rows)
PyObject* py_paged_key_sums(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 9 && sums_call, "paged_key_sums takes nine arguments, and the library's entry points");
  Cache cache;
  Index index;
  const Tensor* sums = plain_tensor(args[4]);
  if (!cache.take(args) || !sums || !index.take(args + 5, cache.k->device())) Py_RETURN_NOTIMPLEMENTED;
  const int64_t rows = PyLong_AsLongLong(args[8]);
  if (PyErr_Occurred()) return nullptr;
  const Tensor& k = *cache.k;
  if (sums->scalar_type() != at::kFloat || sums->dim() != 3 || sums->size(0) != k.size(0) || sums->size(1) != k.size(1) ||
      sums->size(2) != k.size(3) || sums->device() != k.device() || !sums->is_contiguous() || !aligned(*sums, 16) ||
      wants_derivative(*sums) || rows < 1 || rows >= (1 << 30))
    Py_RETURN_NOTIMPLEMENTED;
  {
    const Tensor kp = k, to = *sums, table = *index.table, lengths = *index.lengths, cu = *index.cu;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(kp.device());
    check(sums_call(pointer(kp), (const float*)pointer(cache.k_scales), (float*)to.mutable_data_ptr(), (const int32_t*)pointer(table),
                    (const int32_t*)pointer(lengths), (const int32_t*)pointer(cu), rows, (int)table.size(0), (int)kp.size(1),
                    (int)kp.size(3), (int)kp.size(2), kp.size(0), table.size(1), table.stride(0), cache.k_scales.defined(),
                    cache.k_scales.defined() ? 0 : type_code(kp), stream_of(kp)),
          "moba_paged_key_sums");
    written(to);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// paged_select_blocks(query, sums, page_table, lengths, cu_new, page_size, block_size, topk)
PyObject* py_paged_select_blocks(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 8 && select_call, "paged_select_blocks takes eight arguments, and the library's entry points");
  Index index;
  const Tensor *query = plain_tensor(args[0]), *sums = plain_tensor(args[1]);
  if (!query || !sums || !query->is_cuda() || !index.take(args + 2, query->device()) || wants_derivative(*query) || wants_derivative(*sums) ||
      !half_type(*query) || query->dim() != 3 || sums->scalar_type() != at::kFloat || sums->dim() != 3 || sums->size(0) < 1 ||
      sums->size(1) < 1 || sums->size(1) > 65535 || sums->size(2) != query->size(2) || (sums->size(2) != 64 && sums->size(2) != 128) ||
      sums->device() != query->device() || !sums->is_contiguous() || !aligned(*sums, 16))
    Py_RETURN_NOTIMPLEMENTED;
  int64_t number[3];
  for (int i = 0; i < 3; ++i) {
    number[i] = PyLong_AsLongLong(args[5 + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  const int64_t page = number[0], block_size = number[1], topk = number[2], hkv = sums->size(1);
  int64_t strides[3];
  if (!query_fits(*query, hkv, strides) || page < 16 || page > 256 || (page & (page - 1)) || block_size < 1 || block_size > (1 << 24) ||
      block_size % page || topk < 1 || topk > 64 || index.table->size(1) > kMostBlocks * (block_size / page))
    Py_RETURN_NOTIMPLEMENTED;
  strides[2] = index.table->stride(0);
  Tensor out;
  {
    const Tensor q = *query, s = *sums, table = *index.table, lengths = *index.lengths, cu = *index.cu;
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(q.device());
    const int b = (int)table.size(0), h = (int)q.size(1);
    out = fresh({q.size(0), q.size(1), topk}, at::kInt, q.device());
    Tensor space = bytes(select_bytes(q.size(0), b, h, (int)hkv, (int)page, table.size(1), (int)block_size), q.device());
    check(select_call(pointer(q), (const float*)pointer(s), (int32_t*)mutable_pointer(out), (const int32_t*)pointer(table),
                      (const int32_t*)pointer(lengths), (const int32_t*)pointer(cu), mutable_pointer(space), q.size(0), b, h, (int)hkv,
                      (int)q.size(2), (int)page, s.size(0), table.size(1), (int)block_size, (int)topk, strides, type_code(q), stream_of(q)),
          "moba_paged_select_blocks");
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

namespace {

// The pool and the tables, which the calls write: free_pages, free_count, page_table, lengths, and a number for every sequence
struct Tables {
  Tensor free_pages, free_count, table, lengths, asked;
  int64_t page;
  bool take(PyObject* const* args, PyObject* page_size) {
    Tensor* const to[5] = {&free_pages, &free_count, &table, &lengths, &asked};
    for (int i = 0; i < 5; ++i) {
      const Tensor* t = plain_tensor(args[i]);
      if (!t || t->scalar_type() != at::kInt || !t->is_cuda()) return false;
      *to[i] = *t;
    }
    page = PyLong_AsLongLong(page_size);
    if (PyErr_Occurred()) return false;
    const auto device = free_pages.device();
    for (const Tensor* t : {&free_pages, &free_count, &lengths, &asked})
      if (t->dim() != 1 || !t->is_contiguous() || t->device() != device) return false;
    const int64_t b = lengths.size(0);
    return table.device() == device && free_count.size(0) == 1 && free_pages.size(0) > 0 && free_pages.size(0) <= INT32_MAX && b > 0 &&
           b <= 8192 && asked.size(0) == b && table.dim() == 2 && table.size(0) == b && table.size(1) > 0 && table.numel() <= INT32_MAX &&
           (b == 1 || table.stride(0) >= table.size(1)) && (table.size(1) == 1 || table.stride(1) == 1) && page >= 16 && page <= 256 && !(page & (page - 1));
  }
  int32_t* of(const Tensor& t) const { return (int32_t*)t.mutable_data_ptr(); }
};

}  // namespace

// paged_reserve(free_pages, free_count, page_table, lengths, new_tokens, rows, page_size)
PyObject* py_paged_reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 7 && reserve_call, "paged_reserve takes seven arguments, and the library's entry points");
  Tables t;
  const int64_t rows = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!t.take(args, args[6]) || rows < 0 || rows >= (1 << 30)) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NOTIMPLEMENTED;
  }
  const auto device = t.lengths.device();
  Tensor out[4];
  {
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(device);
    const int64_t b = t.lengths.size(0);
    out[0] = fresh({b + 1}, at::kInt, device);
    out[1] = fresh({rows}, at::kInt, device);
    out[2] = fresh({rows}, at::kInt, device);
    out[3] = fresh({rows}, at::kLong, device);
    const size_t need = reserve_bytes((int)b, rows);
    Tensor space;
    if (need) space = bytes(need, device);
    check(reserve_call(t.of(t.free_pages), t.of(t.free_count), t.of(t.table), t.of(t.lengths), t.of(t.asked), t.of(out[0]), t.of(out[1]),
                       t.of(out[2]), (int64_t*)out[3].mutable_data_ptr(), mutable_pointer(space), (int)b, rows, (int)t.page,
                       t.free_pages.size(0), t.table.size(1), t.table.stride(0), stream_of(t.lengths)),
          "moba_paged_reserve");
    for (const Tensor& x : {t.free_count, t.table, t.lengths}) written(x);
  }
  PyObject* const result = PyTuple_New(4);
  for (int i = 0; result && i < 4; ++i) {
    PyObject* const x = THPVariable_Wrap(std::move(out[i]));
    if (!x) {
      Py_DECREF(result);
      return nullptr;
    }
    PyTuple_SET_ITEM(result, i, x);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

// paged_release(free_pages, free_count, page_table, lengths, keep, page_size)
PyObject* py_paged_release(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6 && release_call, "paged_release takes six arguments, and the library's entry points");
  Tables t;
  if (!t.take(args, args[5])) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NOTIMPLEMENTED;
  }
  {
    const NoGil no_gil;
    const c10::OptionalDeviceGuard guard(t.lengths.device());
    check(release_call(t.of(t.free_pages), t.of(t.free_count), t.of(t.table), t.of(t.lengths), t.of(t.asked), (int)t.lengths.size(0),
                       (int)t.page, t.free_pages.size(0), t.table.size(1), t.table.stride(0), stream_of(t.lengths)),
          "moba_paged_release");
    for (const Tensor& x : {t.free_pages, t.free_count, t.table, t.lengths}) written(x);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// bind_serving(addresses of moba_paged_prefix_attention, .._workspace_bytes, moba_paged_block_attention, .._workspace_bytes,
// moba_paged_key_sums, moba_paged_select_blocks, .._workspace_bytes, moba_paged_reserve, .._workspace_bytes, moba_paged_release), of the
// library whose version bind() has checked
PyObject* py_bind_serving(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "bind_serving takes ten addresses");
  void* at[10];
  for (int i = 0; i < 10; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  prefix_call = reinterpret_cast<decltype(prefix_call)>(at[0]);
  prefix_bytes = reinterpret_cast<decltype(prefix_bytes)>(at[1]);
  block_call = reinterpret_cast<decltype(block_call)>(at[2]);
  block_bytes = reinterpret_cast<decltype(block_bytes)>(at[3]);
  sums_call = reinterpret_cast<decltype(sums_call)>(at[4]);
  select_call = reinterpret_cast<decltype(select_call)>(at[5]);
  select_bytes = reinterpret_cast<decltype(select_bytes)>(at[6]);
  reserve_call = reinterpret_cast<decltype(reserve_call)>(at[7]);
  reserve_bytes = reinterpret_cast<decltype(reserve_bytes)>(at[8]);
  release_call = reinterpret_cast<decltype(release_call)>(at[9]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
