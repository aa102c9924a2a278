// Python binding of the paged calls: from torch tensors to an argument block of
// include/fa_paged_sm100.h and a launch on the current stream, without Python in between.
//
// A decoding step's kernels take a few microseconds, and reading shapes, strides and addresses of
// nine tensors from Python alone takes three times that.  The functions here do the same checks as
// paged.py on the tensors themselves.  What does not pass, or needs more than a launch (a copy of
// unaligned rows, the first use of a device), comes back as None, and paged.py says what is wrong
// or prepares it.  The C ABI is called through the addresses that paged.py hands over, so this
// module needs no link against the library.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/fa_paged_sm100.h"

namespace {

using Tensor = at::Tensor;

int (*g_attn)(const FaPagedAttnArgs*, void*) = nullptr;
int (*g_write)(const FaPagedCopyArgs*, void*) = nullptr;
int (*g_read)(const FaPagedCopyArgs*, void*) = nullptr;
int64_t (*g_workspace)(const FaPagedAttnArgs*) = nullptr;
int (*g_prefix)(const FaPagedPrefixArgs*, void*) = nullptr;
int64_t (*g_prefix_workspace)(const FaPagedPrefixArgs*) = nullptr;
int (*g_weights)(const FaPagedWeightsArgs*, void*) = nullptr;
int64_t (*g_weights_workspace)(const FaPagedWeightsArgs*) = nullptr;
int (*g_evict)(const FaPagedEvictArgs*, void*) = nullptr;
int64_t (*g_evict_workspace)(const FaPagedEvictArgs*) = nullptr;

constexpr int kDevices = 64;
// Devices that paged.py has prepared, and their status words.
bool g_ready[kDevices] = {};
int32_t* g_status[kDevices] = {};

const Tensor* tensor_of(PyObject* x) {
  return THPVariable_Check(x) ? &THPVariable_Unpack(x) : nullptr;
}

// A tensor on device `index` with memory of its own that holds its values (not their negatives, which
// the imaginary part of a conjugate view is).
bool plain(const Tensor& t, int index) {
  return t.is_cuda() && t.get_device() == index && t.layout() == c10::kStrided &&
         t.unsafeGetTensorImpl()->has_storage() && !t.is_neg() &&
         !t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python);
}

// Unit inner stride, and 16-byte strides and address.
bool aligned(const Tensor& t) {
  const int64_t n = t.dim(), eb = t.element_size();
  if (t.size(n - 1) > 1 && t.stride(n - 1) != 1) return false;
  for (int64_t d = 0; d + 1 < n; ++d)
    if (t.size(d) > 1 && (t.stride(d) <= 0 || t.stride(d) * eb % 16)) return false;
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

// Strides of the outer dimensions, a contiguous one where a dimension of size 1 has any.
void strides(const Tensor& t, int64_t* out) {
  const int64_t n = t.dim();
  int64_t inner = t.size(n - 1);
  for (int64_t d = n - 2; d >= 0; --d) {
    out[d] = t.size(d) > 1 ? t.stride(d) : inner;
    inner = std::max(inner, out[d] * t.size(d));
  }
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return FA_DTYPE_FP16;
    case at::kBFloat16: return FA_DTYPE_BF16;
    case at::kFloat8_e4m3fn: return FA_DTYPE_FP8_E4M3;
    default: return -1;
  }
}

struct CacheArgs {
  PyObject *k, *v, *table, *offsets, *lens, *k_scale, *v_scale;
};

bool ints(const Tensor* t, int index) {
  return t && plain(*t, index) && t->scalar_type() == at::kInt;
}

// The sequences of a cache on device `index` (a call without packed rows has no offsets: null); false if
// they are not in order.
bool fill_seqs(const CacheArgs& a, FaPagedCache& c, int index) {
  const Tensor *table = tensor_of(a.table), *lens = tensor_of(a.lens);
  if (!ints(table, index) || !ints(lens, index) || table->dim() != 2 || lens->dim() != 1) return false;
  c.seqs = table->size(0);
  c.table_cols = table->size(1);
  if (lens->size(0) != c.seqs || !lens->is_contiguous() || (c.table_cols > 1 && table->stride(1) != 1))
    return false;
  if (a.offsets) {
    const Tensor* offsets = tensor_of(a.offsets);
    if (!ints(offsets, index) || offsets->dim() != 1 || offsets->size(0) != c.seqs + 1 ||
        !offsets->is_contiguous())
      return false;
    c.offsets = static_cast<const int32_t*>(offsets->const_data_ptr());
  }
  c.table_stride = c.seqs > 1 ? table->stride(0) : c.table_cols;
  c.page_table = static_cast<const int32_t*>(table->const_data_ptr());
  c.kv_lens = static_cast<const int32_t*>(lens->const_data_ptr());
  return true;
}

// The cache and its sequences; false if they are not in order (the sizes are left to the library).
bool fill_cache(const CacheArgs& a, FaPagedCache& c, int& index) {
  const Tensor *k = tensor_of(a.k), *v = tensor_of(a.v);
  if (!k || !v || !k->is_cuda()) return false;
  index = k->get_device();
  if (index < 0 || index >= kDevices || !g_ready[index]) return false;
  for (const Tensor* t : {k, v})
    if (!plain(*t, index)) return false;
  if (!fill_seqs(a, c, index)) return false;
  c.dtype = code_of(k->scalar_type());
  if (c.dtype < 0 || k->scalar_type() != v->scalar_type() || k->dim() != 4 ||
      k->sizes() != v->sizes() || !aligned(*k) || !aligned(*v))
    return false;
  c.num_pages = k->size(0);
  c.heads_kv = k->size(1);
  c.page_size = k->size(2);
  c.head_dim = k->size(3);
  if (c.num_pages < 1 || c.heads_kv < 1 || c.page_size < 8 || c.page_size > 1024 ||
      (c.page_size & (c.page_size - 1)))
    return false;
  strides(*k, c.k_stride);
  strides(*v, c.v_stride);
  c.k = const_cast<void*>(k->const_data_ptr());
  c.v = const_cast<void*>(v->const_data_ptr());
  if ((c.dtype == FA_DTYPE_FP8_E4M3) != (a.k_scale != Py_None) ||
      (a.k_scale != Py_None) != (a.v_scale != Py_None))
    return false;
  if (a.k_scale != Py_None) {
    const Tensor *ks = tensor_of(a.k_scale), *vs = tensor_of(a.v_scale);
    if (!ks || !vs) return false;
    for (const Tensor* t : {ks, vs})
      if (!plain(*t, index) || t->scalar_type() != at::kFloat ||
          t->sizes() != k->sizes().slice(0, 3) || !aligned(*t))
        return false;
    strides(*ks, c.k_scale_stride);
    strides(*vs, c.v_scale_stride);
    c.k_scale = static_cast<float*>(const_cast<void*>(ks->const_data_ptr()));
    c.v_scale = static_cast<float*>(const_cast<void*>(vs->const_data_ptr()));
  }
  return true;
}

// Packed rows [total, heads, head_dim] that go with the cache.
bool rows_ok(const Tensor* t, const FaPagedCache& c, int index) {
  if (!t || !plain(*t, index) || t->dim() != 3 || t->size(2) != c.head_dim || !aligned(*t))
    return false;
  const int code = code_of(t->scalar_type());
  return (code == FA_DTYPE_FP16 || code == FA_DTYPE_BF16) &&
         (code == c.dtype || c.dtype == FA_DTYPE_FP8_E4M3);
}

// A tensor given by the caller was written: autograd has to know, as of any operation in place.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* none() { Py_RETURN_NONE; }

// An upper bound given as an integer or None (0).
bool fill_bound(PyObject* a, int64_t& out) {
  if (a == Py_None) return true;
  out = PyLong_Check(a) ? PyLong_AsLongLong(a) : -1;
  if (out >= 0) return true;
  PyErr_Clear();
  return false;
}

// What attention calls have in common; false if it is not in order.
bool fill_attention(const Tensor* q, const CacheArgs& cache, PyObject* causal, PyObject* sm_scale,
                    PyObject* max_q_len, FaPagedAttnArgs& x, int& index) {
  x.struct_size = sizeof(x);
  if (!fill_cache(cache, x.cache, index) || !rows_ok(q, x.cache, index)) return false;
  x.total = q->size(0);
  x.heads_q = q->size(1);
  if (x.heads_q < 1 || x.heads_q % x.cache.heads_kv) return false;
  x.dtype = code_of(q->scalar_type());
  x.causal = PyObject_IsTrue(causal);
  const double scale = PyFloat_AsDouble(sm_scale);
  if (x.causal < 0 || (scale == -1.0 && PyErr_Occurred())) {
    PyErr_Clear();
    return false;
  }
  x.sm_scale = static_cast<float>(scale);
  return fill_bound(max_q_len, x.max_q_len);
}

// The tensors that an attention call writes: given (not None) or new; false if they are not in order.
bool fill_outputs(const Tensor* q, PyObject* out_arg, PyObject* lse_arg, FaPagedAttnArgs& x, int index,
                  Tensor& out, Tensor& lse) {
  if (out_arg != Py_None) {
    const Tensor* t = tensor_of(out_arg);
    if (!t || !plain(*t, index) || t->sizes() != q->sizes() ||
        t->scalar_type() != q->scalar_type() || !aligned(*t))
      return false;
    out = *t;
  } else {
    out = at::empty_like(*q);
    if (!aligned(out)) return false;
  }
  if (lse_arg != Py_None) {
    const Tensor* t = tensor_of(lse_arg);
    if (!t || !plain(*t, index) || t->dim() != 2 || t->size(0) != x.total ||
        t->size(1) != x.heads_q || t->scalar_type() != at::kFloat || !t->is_contiguous())
      return false;
    lse = *t;
  } else {
    lse = at::empty({x.total, x.heads_q}, q->options().dtype(at::kFloat));
  }
  strides(*q, x.q_stride);
  strides(out, x.o_stride);
  x.q = q->const_data_ptr();
  x.o = out.mutable_data_ptr();
  x.lse = static_cast<float*>(lse.mutable_data_ptr());
  x.dev_status = g_status[index];
  return true;
}

PyObject* outputs(PyObject* out_arg, PyObject* lse_arg, Tensor& out, Tensor& lse) {
  if (out_arg != Py_None) written(out);
  if (lse_arg != Py_None) written(lse);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
  return r;
}

// attention(q, k_cache, v_cache, page_table, offsets, kv_lens, causal, sm_scale, k_scale, v_scale,
//           max_q_len, out, lse) -> (out, lse), a status code, or None
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) return none();
  FaPagedAttnArgs x{};
  int index = -1;
  const Tensor* q = tensor_of(a[0]);
  if (!fill_attention(q, {a[1], a[2], a[3], a[4], a[5], a[8], a[9]}, a[6], a[7], a[10], x, index))
    return none();
  const c10::cuda::OptionalCUDAGuard guard(q->device());
  Tensor out, lse;
  if (!fill_outputs(q, a[11], a[12], x, index, out, lse)) return none();
  if (x.total > 0 && x.cache.seqs > 0) {
    x.workspace_bytes = g_workspace(&x);
    if (x.workspace_bytes < 0) return none();
    // freed when this returns, in the order of the current stream
    const c10::DataPtr workspace =
        c10::cuda::CUDACachingAllocator::get()->allocate(x.workspace_bytes);
    x.workspace = workspace.get();
    const int rc = g_attn(&x, c10::cuda::getCurrentCUDAStream(index).stream());
    if (rc != FA_OK) return PyLong_FromLong(rc);
  }
  return outputs(a[11], a[12], out, lse);
  END_HANDLE_TH_ERRORS
}

// prefix_attention(q, k_cache, v_cache, prefix_table, prefix_offsets, prefix_lens, page_table, offsets,
//                  kv_lens, causal, sm_scale, k_scale, v_scale, max_q_len, max_prefix_q_len, out, lse)
//   -> (out, lse), a status code, or None
PyObject* prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 17) return none();
  FaPagedPrefixArgs x{};
  x.struct_size = sizeof(x);
  int index = -1;
  const Tensor* q = tensor_of(a[0]);
  // the prefixes first: they are sequences of the same cache
  if (!fill_attention(q, {a[1], a[2], a[3], a[4], a[5], a[11], a[12]}, a[9], a[10], a[14], x.attn, index))
    return none();
  x.prefix_table = x.attn.cache.page_table;
  x.prefix_offsets = x.attn.cache.offsets;
  x.prefix_lens = x.attn.cache.kv_lens;
  x.prefix_stride = x.attn.cache.table_stride;
  x.prefix_cols = x.attn.cache.table_cols;
  x.prefixes = x.attn.cache.seqs;
  x.max_prefix_q_len = x.attn.max_q_len;
  x.attn.max_q_len = 0;
  if (!fill_seqs({a[1], a[2], a[6], a[7], a[8], a[11], a[12]}, x.attn.cache, index) ||
      !fill_bound(a[13], x.attn.max_q_len))
    return none();
  const c10::cuda::OptionalCUDAGuard guard(q->device());
  Tensor out, lse;
  if (!fill_outputs(q, a[15], a[16], x.attn, index, out, lse)) return none();
  if (x.attn.total > 0 && x.attn.cache.seqs > 0) {
    x.attn.workspace_bytes = g_prefix_workspace(&x);
    if (x.attn.workspace_bytes < 0) return none();
    const c10::DataPtr workspace =
        c10::cuda::CUDACachingAllocator::get()->allocate(x.attn.workspace_bytes);
    x.attn.workspace = workspace.get();
    const int rc = g_prefix(&x, c10::cuda::getCurrentCUDAStream(index).stream());
    if (rc != FA_OK) return PyLong_FromLong(rc);
  }
  return outputs(a[15], a[16], out, lse);
  END_HANDLE_TH_ERRORS
}

// read_new(total, dtype code, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
//   -> (k, v), a status code, or None
PyObject* read_new(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !PyLong_Check(a[0]) || !PyLong_Check(a[1])) return none();
  FaPagedCopyArgs x{};
  x.struct_size = sizeof(x);
  int index = -1;
  if (!fill_cache({a[2], a[3], a[4], a[5], a[6], a[7], a[8]}, x.cache, index)) return none();
  x.total = PyLong_AsLongLong(a[0]);
  x.dtype = static_cast<int32_t>(PyLong_AsLong(a[1]));
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (x.total < 0 || (x.dtype != FA_DTYPE_FP16 && x.dtype != FA_DTYPE_BF16) ||
      (x.dtype != x.cache.dtype && x.cache.dtype != FA_DTYPE_FP8_E4M3))
    return none();
  const Tensor& cache = *tensor_of(a[2]);
  const c10::cuda::OptionalCUDAGuard guard(cache.device());
  const auto options =
      cache.options().dtype(x.dtype == FA_DTYPE_FP16 ? at::kHalf : at::kBFloat16);
  Tensor k = at::empty({x.total, x.cache.heads_kv, x.cache.head_dim}, options);
  Tensor v = at::empty({x.total, x.cache.heads_kv, x.cache.head_dim}, options);
  strides(k, x.k_stride);
  strides(v, x.v_stride);
  x.k = k.mutable_data_ptr();
  x.v = v.mutable_data_ptr();
  x.dev_status = g_status[index];
  const int rc = g_read(&x, c10::cuda::getCurrentCUDAStream(index).stream());
  if (rc != FA_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
  return r;
  END_HANDLE_TH_ERRORS
}

// copy(write, k, v, k_cache, v_cache, page_table, offsets, kv_lens, k_scale, v_scale)
//   -> status code, or None
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) return none();
  FaPagedCopyArgs x{};
  x.struct_size = sizeof(x);
  int index = -1;
  const Tensor *k = tensor_of(a[1]), *v = tensor_of(a[2]);
  if (!fill_cache({a[3], a[4], a[5], a[6], a[7], a[8], a[9]}, x.cache, index) ||
      !rows_ok(k, x.cache, index) || !rows_ok(v, x.cache, index) || k->sizes() != v->sizes() ||
      k->scalar_type() != v->scalar_type() || k->size(1) != x.cache.heads_kv)
    return none();
  x.total = k->size(0);
  x.dtype = code_of(k->scalar_type());
  strides(*k, x.k_stride);
  strides(*v, x.v_stride);
  x.k = const_cast<void*>(k->const_data_ptr());
  x.v = const_cast<void*>(v->const_data_ptr());
  x.dev_status = g_status[index];
  const c10::cuda::OptionalCUDAGuard guard(k->device());
  void* stream = c10::cuda::getCurrentCUDAStream(index).stream();
  const bool write = a[0] == Py_True;
  const int rc = write ? g_write(&x, stream) : g_read(&x, stream);
  if (rc == FA_OK)
    for (int i : {write ? 3 : 1, write ? 4 : 2, write ? 8 : 0, write ? 9 : 0})
      if (i > 0 && a[i] != Py_None) written(*tensor_of(a[i]));
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// One float for each (page, head, row) of the cache.
bool per_token(const Tensor* t, const Tensor& cache, int index) {
  return t && plain(*t, index) && t->scalar_type() == at::kFloat &&
         t->sizes() == cache.sizes().slice(0, 3) && aligned(*t);
}

// weights(q, lse, k_cache, page_table, offsets, kv_lens, weights, causal, sm_scale, k_scale, max_q_len,
//         reset_new) -> status code, or None
PyObject* weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) return none();
  FaPagedAttnArgs y{};
  int index = -1;
  const Tensor *q = tensor_of(a[0]), *lse = tensor_of(a[1]), *out = tensor_of(a[6]);
  // (there are no values: the keys stand for them)
  if (!fill_attention(q, {a[2], a[2], a[3], a[4], a[5], a[9], a[9]}, a[7], a[8], a[10], y, index) ||
      !per_token(out, *tensor_of(a[2]), index))
    return none();
  if (!lse || !plain(*lse, index) || lse->dim() != 2 || lse->size(0) != y.total || lse->size(1) != y.heads_q ||
      lse->scalar_type() != at::kFloat || !lse->is_contiguous())
    return none();
  FaPagedWeightsArgs x{};
  x.struct_size = sizeof(x);
  x.q = q->const_data_ptr();
  x.lse = static_cast<const float*>(lse->const_data_ptr());
  x.weights = static_cast<float*>(const_cast<void*>(out->const_data_ptr()));
  x.dev_status = g_status[index];
  x.cache = y.cache;
  strides(*q, x.q_stride);
  strides(*out, x.weights_stride);
  x.total = y.total;
  x.heads_q = y.heads_q;
  x.max_q_len = y.max_q_len;
  x.dtype = y.dtype;
  x.causal = y.causal;
  x.reset_new = a[11] == Py_True;
  x.sm_scale = y.sm_scale;
  if (x.total > 0 && x.cache.seqs > 0) {
    const c10::cuda::OptionalCUDAGuard guard(q->device());
    x.workspace_bytes = g_weights_workspace(&x);
    if (x.workspace_bytes < 0) return none();
    const c10::DataPtr workspace =
        c10::cuda::CUDACachingAllocator::get()->allocate(x.workspace_bytes);
    x.workspace = workspace.get();
    const int rc = g_weights(&x, c10::cuda::getCurrentCUDAStream(index).stream());
    if (rc != FA_OK) return PyLong_FromLong(rc);
    written(*out);
  }
  return PyLong_FromLong(FA_OK);
  END_HANDLE_TH_ERRORS
}

// evict(k_cache, v_cache, weights, page_table, kv_lens, keep, recent, k_scale, v_scale, to_table)
//   -> (new_lens, kept), a status code, or None
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 || !PyLong_Check(a[5]) || !PyLong_Check(a[6])) return none();
  FaPagedEvictArgs x{};
  x.struct_size = sizeof(x);
  int index = -1;
  if (!fill_cache({a[0], a[1], a[3], nullptr, a[4], a[7], a[8]}, x.cache, index)) return none();
  const Tensor& cache = *tensor_of(a[0]);
  const Tensor* weights = tensor_of(a[2]);
  if (!per_token(weights, cache, index)) return none();
  x.keep = PyLong_AsLongLong(a[5]);
  x.recent = PyLong_AsLongLong(a[6]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (x.keep < 0 || x.keep > (1 << 30) || x.recent < 0 || x.recent > x.keep) return none();
  x.in_place = a[9] == Py_None;
  if (!x.in_place) {
    const Tensor* to = tensor_of(a[9]);
    if (!ints(to, index) || to->dim() != 2 || to->size(0) != x.cache.seqs ||
        (to->size(1) > 1 && to->stride(1) != 1))
      return none();
    x.to_cols = to->size(1);
    x.to_stride = x.cache.seqs > 1 ? to->stride(0) : x.to_cols;
    x.to_table = static_cast<const int32_t*>(to->const_data_ptr());
  }
  const c10::cuda::OptionalCUDAGuard guard(cache.device());
  strides(*weights, x.weights_stride);
  x.workspace_bytes = g_evict_workspace(&x);
  if (x.workspace_bytes < 0) return none();
  const auto options = cache.options().dtype(at::kInt);
  Tensor lens = at::empty({x.cache.seqs}, options);
  Tensor kept = at::empty({x.cache.seqs, x.cache.heads_kv, x.keep}, options);
  x.weights = static_cast<float*>(const_cast<void*>(weights->const_data_ptr()));
  x.new_lens = static_cast<int32_t*>(lens.mutable_data_ptr());
  x.kept = static_cast<int32_t*>(kept.mutable_data_ptr());
  x.dev_status = g_status[index];
  const c10::DataPtr workspace = c10::cuda::CUDACachingAllocator::get()->allocate(x.workspace_bytes);
  x.workspace = workspace.get();
  const int rc = g_evict(&x, c10::cuda::getCurrentCUDAStream(index).stream());
  if (rc != FA_OK) return PyLong_FromLong(rc);
  for (int i : {0, 1, 2, 7, 8})
    if (a[i] != Py_None) written(*tensor_of(a[i]));
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(lens)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(kept)));
  return r;
  END_HANDLE_TH_ERRORS
}

// setup(attention, workspace_bytes, write, read): addresses of the C ABI
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kCalls = 4;
  void* p[kCalls];
  if (n != kCalls) return none();
  for (int i = 0; i < kCalls; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : none();
  }
  g_attn = reinterpret_cast<decltype(g_attn)>(p[0]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[1]);
  g_write = reinterpret_cast<decltype(g_write)>(p[2]);
  g_read = reinterpret_cast<decltype(g_read)>(p[3]);
  return PyBool_FromLong(1);
}

// setup_more(prefix attention, weights, evict, each with its workspace_bytes): those of the other calls
PyObject* setup_more(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kCalls = 6;
  void* p[kCalls];
  if (n != kCalls) return none();
  for (int i = 0; i < kCalls; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : none();
  }
  g_prefix = reinterpret_cast<decltype(g_prefix)>(p[0]);
  g_prefix_workspace = reinterpret_cast<decltype(g_prefix_workspace)>(p[1]);
  g_weights = reinterpret_cast<decltype(g_weights)>(p[2]);
  g_weights_workspace = reinterpret_cast<decltype(g_weights_workspace)>(p[3]);
  g_evict = reinterpret_cast<decltype(g_evict)>(p[4]);
  g_evict_workspace = reinterpret_cast<decltype(g_evict_workspace)>(p[5]);
  return PyBool_FromLong(1);
}

// set_status(device index, address of its status word or 0, whether calls may use the device)
PyObject* set_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) return none();
  const long index = PyLong_AsLong(a[0]);
  void* p = PyLong_AsVoidPtr(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if (index >= 0 && index < kDevices && g_attn) {
    g_status[index] = static_cast<int32_t*>(p);
    g_ready[index] = a[2] == Py_True;
  }
  return none();
}

PyMethodDef methods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {"prefix_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prefix_attention)), METH_FASTCALL, nullptr},
    {"weights", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(weights)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(evict)), METH_FASTCALL, nullptr},
    {"read_new", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(read_new)), METH_FASTCALL, nullptr},
    {"copy", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(copy)), METH_FASTCALL, nullptr},
    {"setup", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(setup)), METH_FASTCALL, nullptr},
    {"setup_more", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(setup_more)), METH_FASTCALL, nullptr},
    {"set_status", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(set_status)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_binding() { return PyModule_Create(&module); }
