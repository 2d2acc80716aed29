// _torchcall: the decode call path of lowbit.ops (ops.gemv / ops.linear at versions 5 and 6) as one CPython call
// that takes torch tensors. It unpacks them in C++ (no per-attribute Python calls), checks what the C ABI cannot
// see -- dtype, device, shape, contiguity of x, out and bias, and that x's device is the current one -- allocates
// the output when none is given, and calls the C ABI of liblowbit_b200.so on torch's current stream. Anything
// unusual returns None, and the Python caller then takes its fully checked path (which raises the reference's
// errors); a refusal by the C ABI raises RuntimeError with lb_last_error().
//
//   gemv(x, w_ptr, s_ptr, device, n, k, group, version, out=None, bias=None) -> Tensor | None
//
// and, the same way, the calls of a chunk of new tokens (ops.linear_w8, lowbit.paged):
//   linear_w8(x, q, scales, out, bias) -> Tensor | None   (q, scales: a W8Weight's, its layout)
//   norm_rope_append(qkv, cache_ptr, device, positions, slots, nh, inv_freq, q_norm, k_norm, eps, out) -> Tensor | None
//   paged_attention(q, cache_ptr, device, page_table, seq_lens, cu_new, max_new, max_len, scale, out) -> Tensor | None
//
// and of a step of drafted tokens:
//   linear_f8(x, q, scales, out, bias) -> Tensor | None   (q as bytes, scales: an F8Weight's)
//   paged_tree_attention(q, cache_ptr, device, page_table, seq_lens, cu_new, mask, max_new, max_len, scale, out) -> Tensor | None
//   plan(page_table, seq_lens, new_lens, page_size, tokens, held, free_pages, free_count, parents, max_new) -> tuple | None
//   verify(logits, tokens, parents, cu_new, max_new, max_path, seq_lens) -> tuple | None
//   compact(caches, PagedCache, page_table, seq_lens, cu_new, path, accepted, out) -> Tensor | None
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/TensorImpl.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/lowbit_b200.h"

namespace {

bool half_cuda_on(const at::Tensor& t, int dev) {
  return t.scalar_type() == at::kHalf && t.is_cuda() && t.get_device() == dev && t.is_contiguous();
}

PyObject* tc_gemv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs < 8 || nargs > 10) {
    PyErr_SetString(PyExc_TypeError, "gemv(x, w_ptr, s_ptr, device, n, k, group, version, out=None, bias=None)");
    return nullptr;
  }
  if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
  long long v[7];
  for (int i = 0; i < 7; ++i) {
    v[i] = PyLong_AsLongLong(args[1 + i]);
    if (v[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  const void* w = reinterpret_cast<const void*>(static_cast<uintptr_t>(v[0]));
  const void* s = reinterpret_cast<const void*>(static_cast<uintptr_t>(v[1]));
  const int dev = static_cast<int>(v[2]), version = static_cast<int>(v[6]);
  const int64_t n = v[3], k = v[4], group = v[5];
  PyObject* out_obj = nargs > 8 ? args[8] : Py_None;
  PyObject* bias_obj = nargs > 9 ? args[9] : Py_None;

  const at::Tensor& x = THPVariable_Unpack(args[0]);
  if (!half_cuda_on(x, dev) || x.dim() != 2 || x.size(1) != k || x.size(0) == 0 ||
      c10::cuda::current_device() != dev)
    Py_RETURN_NONE;
  const int64_t m = x.size(0);
  const void* bias = nullptr;
  if (bias_obj != Py_None) {
    if (!THPVariable_Check(bias_obj)) Py_RETURN_NONE;
    const at::Tensor& b = THPVariable_Unpack(bias_obj);
    if (!half_cuda_on(b, dev) || b.dim() != 1 || b.size(0) != n) Py_RETURN_NONE;
    bias = b.data_ptr();
  }
  at::Tensor y;
  if (out_obj == Py_None) {
    y = at::empty({m, n}, x.options());
  } else {
    if (!THPVariable_Check(out_obj)) Py_RETURN_NONE;
    const at::Tensor& o = THPVariable_Unpack(out_obj);
    if (!half_cuda_on(o, dev) || o.dim() != 2 || o.size(0) != m || o.size(1) != n) Py_RETURN_NONE;
    y = o;
  }
  const auto st = reinterpret_cast<lb_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream());
  int rc;
  if (bias)
    rc = lb_w4_linear(x.data_ptr(), w, s, bias, y.data_ptr(), m, n, k, group, version, st);
  else if (version == 5)
    rc = lb_w4_gemm_tc(x.data_ptr(), w, s, y.data_ptr(), m, n, k, group, 0, st);
  else
    rc = lb_w4_gemv(x.data_ptr(), w, s, y.data_ptr(), m, n, k, group, version, 0, st);
  if (rc) {
    const char* msg = lb_last_error();
    PyErr_SetString(PyExc_RuntimeError, (msg && msg[0]) ? msg : lb_status_string(rc));
    return nullptr;
  }
  if (out_obj != Py_None) {
    Py_INCREF(out_obj);
    return out_obj;
  }
  return THPVariable_Wrap(std::move(y));
}

bool to_ints(PyObject* const* args, long long* v, int n) {
  for (int i = 0; i < n; ++i) {
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}

// The tensor of an argument, or null when it is none, or not on that device
const at::Tensor* tensor_on(PyObject* o, long long dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev ? &t : nullptr;
}

lb_stream_t stream_of(long long dev) {
  return reinterpret_cast<lb_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream());
}

PyObject* refused(int rc) {
  const char* msg = lb_last_error();
  PyErr_SetString(PyExc_RuntimeError, (msg && msg[0]) ? msg : lb_status_string(rc));
  return nullptr;
}

PyObject* result(PyObject* out_obj, at::Tensor& y) {
  if (out_obj != Py_None) {
    Py_INCREF(out_obj);
    return out_obj;
  }
  return THPVariable_Wrap(std::move(y));
}

// C++ exceptions (torch's allocator, above all) become Python's
template <PyObject* (*F)(PyObject* const*)>
PyObject* guarded(PyObject* const* args) {
  try {
    return F(args);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* linear_w8(PyObject* const* args) {
  if (!THPVariable_Check(args[1])) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(args[1]);
  if (!q.is_cuda() || q.scalar_type() != at::kChar || q.dim() != 2 || q.stride(1) != 1) Py_RETURN_NONE;
  const long long dev = q.get_device();
  const int64_t n = q.size(0), k = q.size(1), ldw = n > 1 ? q.stride(0) : (k + 15) / 16 * 16;
  const at::Tensor* scales = tensor_on(args[2], dev);
  if (!scales || scales->scalar_type() != at::kFloat || scales->dim() != 1 || scales->size(0) != n ||
      !scales->is_contiguous())
    Py_RETURN_NONE;
  const at::Tensor* x = tensor_on(args[0], dev);
  if (!x || x->dim() != 2 || x->size(1) != k || x->size(0) == 0 || c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
  const int64_t m = x->size(0), ldx = m > 1 ? x->stride(0) : k;
  if (x->stride(1) != 1 || ldx < k) Py_RETURN_NONE;
  const void* bias = nullptr;
  if (args[4] != Py_None) {
    const at::Tensor* b = tensor_on(args[4], dev);
    if (!b || b->scalar_type() != type || b->dim() != 1 || b->size(0) != n || !b->is_contiguous()) Py_RETURN_NONE;
    bias = b->data_ptr();
  }
  at::Tensor y;
  if (args[3] == Py_None) {
    y = at::empty({m, n}, x->options());
  } else {
    const at::Tensor* o = tensor_on(args[3], dev);
    if (!o || o->scalar_type() != type || o->dim() != 2 || o->size(0) != m || o->size(1) != n || !o->is_contiguous())
      Py_RETURN_NONE;
    y = *o;
  }
  const int64_t need = lb_w8_workspace(m, n, k);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, x->options().dtype(at::kByte));
  const int rc = lb_w8_linear(x->data_ptr(), type == at::kHalf ? LB_F16 : LB_BF16, ldx,
                              q.data_ptr(), ldw, scales->data_ptr<float>(), bias, y.data_ptr(), m, n, k,
                              need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  return rc ? refused(rc) : result(args[3], y);
}

PyObject* linear_f8(PyObject* const* args) {
  if (!THPVariable_Check(args[1])) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(args[1]);
  if (!q.is_cuda() || q.scalar_type() != at::kByte || q.dim() != 2 || q.stride(1) != 1) Py_RETURN_NONE;
  const long long dev = q.get_device();
  const int64_t n = q.size(0), k = q.size(1), ldw = n > 1 ? q.stride(0) : (k + 15) / 16 * 16;
  const at::Tensor* scales = tensor_on(args[2], dev);
  if (!scales || scales->scalar_type() != at::kFloat || scales->dim() != 2 || scales->size(0) != (n + 127) / 128 ||
      scales->size(1) != (k + 127) / 128 || !scales->is_contiguous())
    Py_RETURN_NONE;
  const at::Tensor* x = tensor_on(args[0], dev);
  if (!x || x->dim() != 2 || x->size(1) != k || x->size(0) == 0 || c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const auto type = x->scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) Py_RETURN_NONE;
  const int64_t m = x->size(0), ldx = m > 1 ? x->stride(0) : k;
  if (x->stride(1) != 1 || ldx < k) Py_RETURN_NONE;
  const void* bias = nullptr;
  if (args[4] != Py_None) {
    const at::Tensor* b = tensor_on(args[4], dev);
    if (!b || b->scalar_type() != type || b->dim() != 1 || b->size(0) != n || !b->is_contiguous()) Py_RETURN_NONE;
    bias = b->data_ptr();
  }
  at::Tensor y;
  if (args[3] == Py_None) {
    y = at::empty({m, n}, x->options());
  } else {
    const at::Tensor* o = tensor_on(args[3], dev);
    if (!o || o->scalar_type() != type || o->dim() != 2 || o->size(0) != m || o->size(1) != n || !o->is_contiguous())
      Py_RETURN_NONE;
    y = *o;
  }
  const int64_t need = lb_f8_workspace(m, n, k);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, x->options().dtype(at::kByte));
  const int rc = lb_f8_linear(x->data_ptr(), type == at::kHalf ? LB_F16 : LB_BF16, ldx, q.data_ptr(), ldw, scales->data_ptr<float>(),
                              bias, y.data_ptr(), m, n, k, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  return rc ? refused(rc) : result(args[3], y);
}

at::ScalarType cache_type(const lb_paged_cache* c) { return c->dtype == LB_F16 ? at::kHalf : at::kBFloat16; }

// a contiguous vector of that type and length on the device
bool vector_of(const at::Tensor* t, at::ScalarType type, int64_t n) {
  return t && t->scalar_type() == type && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

// `out`: a contiguous [t, nh, hd] tensor, new when none is given; false when what is given is not one
bool heads_out(PyObject* o, long long dev, const at::Tensor& like, int64_t t, int64_t nh, int64_t hd, at::Tensor* y) {
  if (o == Py_None) {
    *y = at::empty({t, nh, hd}, like.options());
    return true;
  }
  const at::Tensor* g = tensor_on(o, dev);
  if (!g || g->scalar_type() != like.scalar_type() || g->dim() != 3 || g->size(0) != t || g->size(1) != nh ||
      g->size(2) != hd || !g->is_contiguous())
    return false;
  *y = *g;
  return true;
}

PyObject* norm_rope_append(PyObject* const* args) {
  long long v[3];
  if (!to_ints(args + 1, v, 2) || !to_ints(args + 5, v + 2, 1)) return nullptr;
  const auto* c = reinterpret_cast<const lb_paged_cache*>(static_cast<uintptr_t>(v[0]));
  const long long dev = v[1], nh = v[2];
  const double eps = PyFloat_AsDouble(args[9]);
  if (eps == -1.0 && PyErr_Occurred()) return nullptr;
  const at::Tensor *x = tensor_on(args[0], dev), *pos = tensor_on(args[3], dev), *slots = tensor_on(args[4], dev),
                   *freq = tensor_on(args[6], dev);
  if (!x || !freq || nh < 1 || nh > 65536 || c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const auto type = cache_type(c);
  const int64_t width = (nh + 2 * (int64_t)c->nkv) * c->hd;
  if (x->scalar_type() != type || x->dim() != 2 || x->size(0) == 0 || x->size(1) != width || x->stride(1) != 1)
    Py_RETURN_NONE;
  const int64_t t = x->size(0), ld = t > 1 ? x->stride(0) : width;
  if (ld % 8 || ld < width || !vector_of(pos, at::kLong, t) || !vector_of(slots, at::kLong, t) ||
      !vector_of(freq, at::kFloat, freq->numel()) || freq->numel() % 8 || 2 * freq->numel() > c->hd)
    Py_RETURN_NONE;
  const void *qn = nullptr, *kn = nullptr;
  if (args[7] != Py_None || args[8] != Py_None) {
    const at::Tensor *a = tensor_on(args[7], dev), *b = tensor_on(args[8], dev);
    if (!vector_of(a, type, c->hd) || !vector_of(b, type, c->hd)) Py_RETURN_NONE;
    qn = a->data_ptr();
    kn = b->data_ptr();
  }
  at::Tensor y;
  if (!heads_out(args[10], dev, *x, t, nh, c->hd, &y)) Py_RETURN_NONE;
  const int rot = (int)(2 * freq->numel());
  const int rc = lb_paged_norm_rope_append(x->data_ptr(), ld, t, (int)nh, qn, kn, (float)eps,
                                           rot ? freq->data_ptr<float>() : nullptr, rot, pos->data_ptr<int64_t>(),
                                           slots->data_ptr<int64_t>(), c, y.data_ptr(), stream_of(dev));
  return rc ? refused(rc) : result(args[10], y);
}

// both attentions; the arguments behind cu_new start at args[more], a tree's mask stands before them
template <bool TREE>
PyObject* attend(PyObject* const* args) {
  constexpr int more = TREE ? 7 : 6;
  long long v[2];
  if (!to_ints(args + 1, v, 2)) return nullptr;
  const auto* c = reinterpret_cast<const lb_paged_cache*>(static_cast<uintptr_t>(v[0]));
  const long long dev = v[1];
  const at::Tensor *q = tensor_on(args[0], dev), *table = tensor_on(args[3], dev), *lens = tensor_on(args[4], dev),
                   *cu = tensor_on(args[5], dev);
  if (!q || !table || c10::cuda::current_device() != dev) Py_RETURN_NONE;
  if (q->scalar_type() != cache_type(c) || q->dim() != 3 || q->size(0) == 0 || q->size(1) == 0 ||
      q->size(1) % c->nkv || q->size(2) != c->hd || q->stride(2) != 1)
    Py_RETURN_NONE;
  if (table->scalar_type() != at::kInt || table->dim() != 2 || table->size(0) == 0 || table->size(1) == 0 ||
      table->stride(1) != 1)
    Py_RETURN_NONE;
  const int64_t t = q->size(0), nh = q->size(1), s = table->size(0), w = table->size(1);
  if (s > INT32_MAX || !vector_of(lens, at::kInt, s) || !vector_of(cu, at::kInt, s + 1)) Py_RETURN_NONE;
  const at::Tensor* mask = nullptr;
  if (TREE) {
    mask = tensor_on(args[6], dev);
    if (!mask || mask->scalar_type() != at::kInt || mask->dim() != 2 || mask->size(0) != t || mask->size(1) == 0 || !mask->is_contiguous())
      Py_RETURN_NONE;
  }
  long long bound[2] = {t, w * c->page_size};
  for (int i = 0; i < 2; ++i)
    if (args[more + i] != Py_None && !to_ints(args + more + i, bound + i, 1)) return nullptr;
  double scale = c->hd == 64 ? 0.125 : 0.08838834764831845;   // 1 / sqrt(hd) of the head dims the kernel takes
  if (args[more + 2] != Py_None) {
    scale = PyFloat_AsDouble(args[more + 2]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  }
  at::Tensor y;
  if (!heads_out(args[more + 3], dev, *q, t, nh, c->hd, &y)) Py_RETURN_NONE;
  const int64_t need = (TREE ? lb_paged_tree_attention_workspace : lb_paged_attention_workspace)(t, (int)nh, c, w, (int)s, bound[0], bound[1]);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, q->options().dtype(at::kByte));
  const int64_t ts = t > 1 ? q->stride(0) : 0, hs = nh > 1 ? q->stride(1) : 0, table_stride = s > 1 ? table->stride(0) : w;
  void* const work = need > 0 ? ws.data_ptr() : nullptr;
  const int rc =
      TREE ? lb_paged_tree_attention(q->data_ptr(), ts, hs, t, (int)nh, c, table->data_ptr<int32_t>(), table_stride, w,
                                     lens->data_ptr<int32_t>(), cu->data_ptr<int32_t>(), (int)s,
                                     reinterpret_cast<const uint32_t*>(mask->data_ptr<int32_t>()), mask->size(1), bound[0], bound[1],
                                     (float)scale, y.data_ptr(), nh * c->hd, work, need, stream_of(dev))
           : lb_paged_attention(q->data_ptr(), ts, hs, t, (int)nh, c, table->data_ptr<int32_t>(), table_stride, w,
                                lens->data_ptr<int32_t>(), cu->data_ptr<int32_t>(), (int)s, bound[0], bound[1], (float)scale,
                                y.data_ptr(), nh * c->hd, work, need, stream_of(dev));
  return rc ? refused(rc) : result(args[more + 3], y);
}

PyObject* tuple_of(std::initializer_list<at::Tensor*> tensors) {   // null or undefined: None
  PyObject* r = PyTuple_New((Py_ssize_t)tensors.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (at::Tensor* t : tensors) {
    PyObject* o;
    if (t && t->defined()) {
      o = THPVariable_Wrap(std::move(*t));
    } else {
      Py_INCREF(Py_None);
      o = Py_None;
    }
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// an int32 page table with contiguous rows that do not overlap
bool page_table_of(const at::Tensor* t) {
  return t && t->scalar_type() == at::kInt && t->dim() == 2 && t->size(0) > 0 && t->size(0) <= INT32_MAX && t->size(1) > 0 &&
         t->stride(1) == 1 && (t->size(0) == 1 || t->stride(0) >= t->size(1));
}

// Several outputs from one allocation, each on a 64-byte boundary (seven of their own cost a call's host time 5 us more)
class Outputs {
 public:
  static int64_t padded(int64_t bytes) { return (bytes + 63) / 64 * 64; }
  Outputs(int64_t bytes, const at::Tensor& like) : base_(at::empty({bytes}, like.options().dtype(at::kByte))) {}
  at::Tensor take(at::ScalarType type, at::IntArrayRef sizes) {
    const auto meta = c10::scalarTypeToTypeMeta(type);
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(base_.storage()), base_.key_set(), meta);
    impl->set_storage_offset(at_ / (int64_t)meta.itemsize());
    impl->set_sizes_contiguous(sizes);
    at_ += padded(impl->numel() * (int64_t)meta.itemsize());
    return at::Tensor(std::move(impl));
  }
  void* rest() { return static_cast<uint8_t*>(base_.data_ptr()) + at_; }

 private:
  at::Tensor base_;
  int64_t at_ = 0;
};

PyObject* plan(PyObject* const* args) {
  if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
  const at::Tensor& table = THPVariable_Unpack(args[0]);
  if (!table.is_cuda() || !page_table_of(&table)) Py_RETURN_NONE;
  const long long dev = table.get_device();
  if (c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const int64_t s = table.size(0), w = table.size(1);
  const at::Tensor *lens = tensor_on(args[1], dev), *fresh = tensor_on(args[2], dev);
  if (!vector_of(lens, at::kInt, s) || !vector_of(fresh, at::kInt, s)) Py_RETURN_NONE;
  long long v[2], most = 0;
  if (!to_ints(args + 3, v, 2)) return nullptr;
  const long long page = v[0], tokens = v[1];
  if (tokens < 1 || page < 1 || page > 65536) Py_RETURN_NONE;
  const at::Tensor *held = nullptr, *list = nullptr, *count = nullptr, *parents = nullptr;
  const bool paging = args[5] != Py_None;
  if (paging != (args[6] != Py_None) || paging != (args[7] != Py_None)) Py_RETURN_NONE;
  if (paging) {
    held = tensor_on(args[5], dev), list = tensor_on(args[6], dev), count = tensor_on(args[7], dev);
    if (!list || list->numel() == 0 || !vector_of(held, at::kInt, s) || !vector_of(list, at::kInt, list->numel()) || !vector_of(count, at::kInt, 1))
      Py_RETURN_NONE;
  }
  int64_t words = 0;
  if (args[8] != Py_None) {
    parents = tensor_on(args[8], dev);
    if (!vector_of(parents, at::kInt, tokens)) Py_RETURN_NONE;
    most = tokens;
    if (args[9] != Py_None && !to_ints(args + 9, &most, 1)) return nullptr;
    if (most < 1 || most > 1024) Py_RETURN_NONE;
    words = (most + 31) / 32;
  }
  Outputs outs(Outputs::padded(4 * (s + 1)) + Outputs::padded(4 * s) + 2 * Outputs::padded(8 * tokens) +
                   (paging ? Outputs::padded(4 * s) + Outputs::padded(4) : 0) + (parents ? Outputs::padded(4 * tokens * words) : 0),
               *lens);
  at::Tensor cu = outs.take(at::kInt, {s + 1}), after = outs.take(at::kInt, {s}), pos = outs.take(at::kLong, {tokens}),
             slots = outs.take(at::kLong, {tokens});
  at::Tensor held_out, count_out, mask;
  if (paging) held_out = outs.take(at::kInt, {s}), count_out = outs.take(at::kInt, {1});
  if (parents) mask = outs.take(at::kInt, {tokens, words});
  const int rc = lb_paged_plan(lens->data_ptr<int32_t>(), fresh->data_ptr<int32_t>(), (int)s, table.data_ptr<int32_t>(),
                               s > 1 ? table.stride(0) : w, w, (int)page, tokens, paging ? held->data_ptr<int32_t>() : nullptr,
                               paging ? list->data_ptr<int32_t>() : nullptr, paging ? list->numel() : 0,
                               paging ? count->data_ptr<int32_t>() : nullptr, parents ? parents->data_ptr<int32_t>() : nullptr, words,
                               cu.data_ptr<int32_t>(), after.data_ptr<int32_t>(), paging ? held_out.data_ptr<int32_t>() : nullptr,
                               paging ? count_out.data_ptr<int32_t>() : nullptr, pos.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                               parents ? reinterpret_cast<uint32_t*>(mask.data_ptr<int32_t>()) : nullptr, stream_of(dev));
  return rc ? refused(rc) : tuple_of({&cu, &after, &pos, &slots, &held_out, &count_out, &mask});
}

PyObject* verify(PyObject* const* args) {
  if (!THPVariable_Check(args[0])) Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  if (!x.is_cuda() || x.dim() != 2 || x.size(0) == 0 || x.size(1) == 0 || x.stride(1) != 1) Py_RETURN_NONE;
  const auto type = x.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) Py_RETURN_NONE;
  const long long dev = x.get_device();
  if (c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const int64_t t = x.size(0), vocab = x.size(1), ld = t > 1 ? x.stride(0) : vocab;
  const at::Tensor *tokens = tensor_on(args[1], dev), *parents = tensor_on(args[2], dev), *cu = tensor_on(args[3], dev);
  if (ld < vocab || !vector_of(tokens, at::kLong, t) || !vector_of(parents, at::kInt, t) || !cu || !vector_of(cu, at::kInt, cu->numel()) || cu->numel() < 2 ||
      cu->numel() > INT32_MAX)
    Py_RETURN_NONE;
  long long bound[2] = {t, 0};
  if (args[4] != Py_None && !to_ints(args + 4, bound, 1)) return nullptr;
  bound[1] = bound[0];
  if (args[5] != Py_None && !to_ints(args + 5, bound + 1, 1)) return nullptr;
  if (bound[0] < 1 || bound[0] > 1024 || bound[1] < 1 || bound[1] > 1024) Py_RETURN_NONE;
  const int64_t s = cu->numel() - 1, need = lb_draft_verify_workspace(t, vocab);
  const at::Tensor* lens = nullptr;
  if (args[6] != Py_None) {
    lens = tensor_on(args[6], dev);
    if (!vector_of(lens, at::kInt, s)) Py_RETURN_NONE;
  }
  Outputs outs(Outputs::padded(4 * s) + Outputs::padded(4 * s * bound[1]) + Outputs::padded(8 * s) + Outputs::padded(8 * t) + need, *cu);
  at::Tensor accepted = outs.take(at::kInt, {s}), path = outs.take(at::kInt, {s, bound[1]}), next = outs.take(at::kLong, {s}),
             targets = outs.take(at::kLong, {t});
  const int rc = lb_draft_verify_planned(x.data_ptr(), type == at::kHalf ? LB_F16 : type == at::kBFloat16 ? LB_BF16 : LB_F32, ld, t, vocab,
                                         tokens->data_ptr<int64_t>(), parents->data_ptr<int32_t>(), cu->data_ptr<int32_t>(),
                                         lens ? lens->data_ptr<int32_t>() : nullptr, (int)s, bound[0], bound[1], accepted.data_ptr<int32_t>(),
                                         path.data_ptr<int32_t>(), next.data_ptr<int64_t>(), targets.data_ptr<int64_t>(), outs.rest(), need,
                                         stream_of(dev));
  return rc ? refused(rc) : tuple_of({&accepted, &path, &next, &targets});
}

PyObject* compact(PyObject* const* args) {
  static PyObject* const name = PyUnicode_InternFromString("_place");
  const bool list = PyList_Check(args[0]);
  if (!list && !PyTuple_Check(args[0])) Py_RETURN_NONE;
  const Py_ssize_t layers = list ? PyList_GET_SIZE(args[0]) : PyTuple_GET_SIZE(args[0]);
  if (layers < 1 || layers > 128) Py_RETURN_NONE;
  const lb_paged_cache* caches[128];
  long long dev = -1;
  for (Py_ssize_t i = 0; i < layers; ++i) {
    PyObject* const one = list ? PyList_GET_ITEM(args[0], i) : PyTuple_GET_ITEM(args[0], i);
    if (reinterpret_cast<PyObject*>(Py_TYPE(one)) != args[1]) Py_RETURN_NONE;
    PyObject* const place = PyObject_GetAttr(one, name);   // (address, device)
    if (!place) return nullptr;
    PyObject* const* v = PyTuple_Check(place) && PyTuple_GET_SIZE(place) == 2 ? &PyTuple_GET_ITEM(place, 0) : nullptr;
    long long at[2] = {0, -1};
    const bool ok = v && to_ints(v, at, 2);
    Py_DECREF(place);
    if (!ok || (i > 0 && at[1] != dev)) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    dev = at[1];
    caches[i] = reinterpret_cast<const lb_paged_cache*>(static_cast<uintptr_t>(at[0]));
  }
  const at::Tensor *table = tensor_on(args[2], dev), *lens = tensor_on(args[3], dev), *cu = tensor_on(args[4], dev), *path = tensor_on(args[5], dev),
                   *accepted = tensor_on(args[6], dev);
  if (!page_table_of(table) || c10::cuda::current_device() != dev) Py_RETURN_NONE;
  const int64_t s = table->size(0), w = table->size(1);
  if (!vector_of(lens, at::kInt, s) || !vector_of(cu, at::kInt, s + 1) || !vector_of(accepted, at::kInt, s) || !path ||
      path->scalar_type() != at::kInt || path->dim() != 2 || path->size(0) != s || path->size(1) == 0 || !path->is_contiguous())
    Py_RETURN_NONE;
  at::Tensor y;
  if (args[7] == Py_None) {
    y = at::empty({s}, lens->options());
  } else {
    const at::Tensor* o = tensor_on(args[7], dev);
    if (!vector_of(o, at::kInt, s)) Py_RETURN_NONE;
    y = *o;
  }
  const int rc = lb_paged_compact(caches, (int)layers, table->data_ptr<int32_t>(), s > 1 ? table->stride(0) : w, w, lens->data_ptr<int32_t>(),
                                  cu->data_ptr<int32_t>(), path->data_ptr<int32_t>(), accepted->data_ptr<int32_t>(), (int)s, path->size(1),
                                  y.data_ptr<int32_t>(), args[7] != Py_None, stream_of(dev));
  return rc ? refused(rc) : result(args[7], y);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %d", N, (int)nargs);
    return nullptr;
  }
  return guarded<F>(args);
}

template <PyObject* (*F)(PyObject* const*), int N>
PyCFunction fastcall() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(call<F, N>));
}

PyMethodDef methods[] = {
    {"linear_w8", fastcall<linear_w8, 5>(), METH_FASTCALL,
     "linear_w8(x, q, scales, out, bias) -> Tensor, or None for the checked path"},
    {"norm_rope_append", fastcall<norm_rope_append, 11>(), METH_FASTCALL,
     "norm_rope_append(qkv, cache_ptr, device, positions, slots, nh, inv_freq, q_norm, k_norm, eps, out) -> Tensor, or "
     "None for the checked path"},
    {"linear_f8", fastcall<linear_f8, 5>(), METH_FASTCALL,
     "linear_f8(x, q, scales, out, bias) -> Tensor, or None for the checked path"},
    {"paged_tree_attention", fastcall<attend<true>, 11>(), METH_FASTCALL,
     "paged_tree_attention(q, cache_ptr, device, page_table, seq_lens, cu_new, mask, max_new, max_len, scale, out) -> Tensor, or "
     "None for the checked path"},
    {"plan", fastcall<plan, 10>(), METH_FASTCALL,
     "plan(page_table, seq_lens, new_lens, page_size, tokens, held, free_pages, free_count, parents, max_new) -> tuple, or None "
     "for the checked path"},
    {"verify", fastcall<verify, 7>(), METH_FASTCALL,
     "verify(logits, tokens, parents, cu_new, max_new, max_path, seq_lens) -> tuple, or None for the checked path"},
    {"compact", fastcall<compact, 8>(), METH_FASTCALL,
     "compact(caches, PagedCache, page_table, seq_lens, cu_new, path, accepted, out) -> Tensor, or None for the checked path"},
    {"paged_attention", fastcall<attend<false>, 10>(), METH_FASTCALL,
     "paged_attention(q, cache_ptr, device, page_table, seq_lens, cu_new, max_new, max_len, scale, out) -> Tensor, or "
     "None for the checked path"},
    {"gemv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(tc_gemv)), METH_FASTCALL,
     "gemv(x, w_ptr, s_ptr, device, n, k, group, version, out=None, bias=None) -> Tensor, or None for the checked "
     "path"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&module); }
