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
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
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

PyObject* paged_attention(PyObject* const* args) {
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
  long long bound[2] = {t, w * c->page_size};
  for (int i = 0; i < 2; ++i)
    if (args[6 + i] != Py_None && !to_ints(args + 6 + i, bound + i, 1)) return nullptr;
  double scale = c->hd == 64 ? 0.125 : 0.08838834764831845;   // 1 / sqrt(hd) of the head dims the kernel takes
  if (args[8] != Py_None) {
    scale = PyFloat_AsDouble(args[8]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  }
  at::Tensor y;
  if (!heads_out(args[9], dev, *q, t, nh, c->hd, &y)) Py_RETURN_NONE;
  const int64_t need = lb_paged_attention_workspace(t, (int)nh, c, w, (int)s, bound[0], bound[1]);
  at::Tensor ws;
  if (need > 0) ws = at::empty({need}, q->options().dtype(at::kByte));
  const int rc = lb_paged_attention(q->data_ptr(), t > 1 ? q->stride(0) : 0, nh > 1 ? q->stride(1) : 0, t, (int)nh, c, table->data_ptr<int32_t>(),
                                    s > 1 ? table->stride(0) : w, w, lens->data_ptr<int32_t>(), cu->data_ptr<int32_t>(),
                                    (int)s, bound[0], bound[1], (float)scale, y.data_ptr(), nh * c->hd,
                                    need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  return rc ? refused(rc) : result(args[9], y);
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
    {"paged_attention", fastcall<paged_attention, 10>(), METH_FASTCALL,
     "paged_attention(q, cache_ptr, device, page_table, seq_lens, cu_new, max_new, max_len, scale, out) -> Tensor, or "
     "None for the checked path"},
    {"gemv", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(tc_gemv)), METH_FASTCALL,
     "gemv(x, w_ptr, s_ptr, device, n, k, group, version, out=None, bias=None) -> Tensor, or None for the checked "
     "path"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchcall(void) { return PyModule_Create(&module); }
