// The ordinary calls of the 4-bit cache's operators and of the block copies, from Python objects to the C ABI.
//
// A small call of these operators is bound by the host, and through ctypes most of that is argument handling.
// Measured on the host, through ctypes and here: decode of one short row 14.7 -> 5.5 us, append 26 -> 10.6, gather
// of one history 13 -> 6.2, a fork's copies 27 -> 4.3.  Each function here does that for the ordinary case (plain CUDA tensors of the
// current device, contiguous where the ABI wants it, every shape and type as it should be) and returns None
// for any other, errors among them: the caller (ops.py) then takes its own path, which handles strides, other
// devices and refusals with their messages.  Nothing is kept between calls.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "mi_kv4.h"

namespace {

using at::Tensor;

// The tensor of a plain CUDA tensor of device `dev`, or null.
const Tensor* plain(PyObject* o, int dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided ? &t : nullptr;
}

const Tensor* longs(PyObject* o, int dev, int64_t dims) {  // contiguous int64
  const Tensor* t = plain(o, dev);
  return t && t->scalar_type() == at::kLong && t->dim() == dims && t->is_contiguous() ? t : nullptr;
}

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MI_F32;
    case at::kBFloat16: return MI_BF16;
    case at::kHalf: return MI_F16;
    default: return -1;
  }
}

// 4-bit pools for this head_dim.
struct Pools {
  const Tensor *k, *v;
  int64_t n, h;
  int bs;
};
bool pools_of(PyObject* k, PyObject* v, int64_t d, int dev, Pools& p) {
  p.k = plain(k, dev);
  p.v = plain(v, dev);
  if (!p.k || !p.v || p.k->scalar_type() != at::kByte || p.v->scalar_type() != at::kByte || p.k->dim() != 3 ||
      p.k->sizes() != p.v->sizes() || !p.k->is_contiguous() || !p.v->is_contiguous())
    return false;
  if (d < MI_KV4_GROUP || d > 256 || d % MI_KV4_GROUP) return false;
  const int64_t page = p.k->size(2), token = d * 5 / 8;
  if (page < token || page % token || page / token > (int64_t(1) << 30)) return false;
  p.n = p.k->size(0);
  p.h = p.k->size(1);
  p.bs = (int)(page / token);
  return p.h > 0 && p.h < (int64_t(1) << 30);
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

PyObject* none() { Py_RETURN_NONE; }

// (query, k_pool, v_pool, block_tables, context_lens, scale) -> out
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 6) return none();
  const int dev = c10::cuda::current_device();
  const Tensor* q = plain(a[0], dev);
  const double scale = PyFloat_AsDouble(a[5]);
  if (scale == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (!q || q->dim() != 3 || !q->is_contiguous()) return none();
  const int64_t b = q->size(0), hq = q->size(1), d = q->size(2);
  Pools p;
  const Tensor* tables = longs(a[3], dev, 2);
  const Tensor* ctx = longs(a[4], dev, 1);
  const int code = dtype_of(*q);
  if (code < 0 || !pools_of(a[1], a[2], d, dev, p) || !tables || !ctx || tables->size(0) != b || ctx->size(0) != b || b < 1 ||
      hq < 1 || hq > (1 << 20) || hq % p.h || tables->size(1) < 1)
    return none();
  const int64_t width = tables->size(1);
  const size_t need = mi_kv4_paged_decode_workspace_size(b, (int)hq, (int)p.h, (int)d, width, p.bs, code);
  Tensor ws;
  char* base = nullptr;
  if (need) {
    ws = at::empty({(int64_t)need + 256}, at::TensorOptions().dtype(at::kByte).device(q->device()));
    base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(ws.data_ptr()) + 255) & ~uintptr_t(255));
  }
  Tensor out = at::empty({b, hq * d}, q->options().requires_grad(false));
  const int64_t q_strides[2] = {hq * d, d};
  const int rc = mi_kv4_paged_decode(q->data_ptr(), q_strides, nullptr, nullptr, nullptr, nullptr, p.k->data_ptr(),
                                     p.v->data_ptr(), p.n, p.bs, (int)p.h, (int)d,
                                     static_cast<const int64_t*>(tables->data_ptr()), width, width,
                                     static_cast<const int64_t*>(ctx->data_ptr()), b, (int)hq, (float)scale,
                                     out.data_ptr(), hq * d, base, need, code, stream_of(dev));
  return rc == MI_OK ? THPVariable_Wrap(std::move(out)) : none();
}

// (key, value, slot_mapping, k_pool, v_pool) -> True: tokens [T, H, D] with unit stride along D
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 5) return none();
  const int dev = c10::cuda::current_device();
  const Tensor *k = plain(a[0], dev), *v = plain(a[1], dev), *slots = longs(a[2], dev, 1);
  if (!k || !v || !slots || k->dim() != 3 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() ||
      k->size(0) < 1 || slots->size(0) > k->size(0) || k->stride(2) != 1 || v->stride(2) != 1)
    return none();
  const int code = dtype_of(*k);
  const int64_t d = k->size(2);
  Pools p;
  if (code < 0 || !pools_of(a[3], a[4], d, dev, p) || k->size(1) != p.h) return none();
  const int64_t ks[3] = {k->stride(0), k->stride(1), 0}, vs[3] = {v->stride(0), v->stride(1), 0};
  const int rc = mi_kv4_scatter(k->data_ptr(), v->data_ptr(), ks, vs, k->size(0), 1, nullptr, nullptr,
                                static_cast<const int64_t*>(slots->data_ptr()), slots->size(0), p.k->data_ptr(),
                                p.v->data_ptr(), p.n, p.bs, (int)p.h, (int)d, code, stream_of(dev));
  if (rc != MI_OK) return none();
  Py_RETURN_TRUE;
}

// (key, value, chunk_lens, start_positions, block_tables, k_pool, v_pool) -> True
PyObject* store_chunks(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 7) return none();
  const int dev = c10::cuda::current_device();
  const Tensor *k = plain(a[0], dev), *v = plain(a[1], dev);
  const Tensor *lens = longs(a[2], dev, 1), *starts = longs(a[3], dev, 1), *tables = longs(a[4], dev, 2);
  if (!k || !v || !lens || !starts || !tables || k->dim() != 4 || k->sizes() != v->sizes() ||
      k->scalar_type() != v->scalar_type() || k->stride(3) != 1 || v->stride(3) != 1)
    return none();
  const int code = dtype_of(*k);
  const int64_t b = k->size(0), d = k->size(3);
  Pools p;
  if (code < 0 || !pools_of(a[5], a[6], d, dev, p) || k->size(1) != p.h || b < 1 || k->size(2) < 1 ||
      lens->size(0) != b || starts->size(0) != b || tables->size(0) != b)
    return none();
  const int rc = mi_kv4_store_chunks(k->data_ptr(), v->data_ptr(), k->strides().data(), v->strides().data(), b, k->size(2),
                                     static_cast<const int64_t*>(lens->data_ptr()),
                                     static_cast<const int64_t*>(starts->data_ptr()),
                                     static_cast<const int64_t*>(tables->data_ptr()), tables->size(1), tables->size(1),
                                     p.k->data_ptr(), p.v->data_ptr(), p.n, p.bs, (int)p.h, (int)d, code, stream_of(dev));
  if (rc != MI_OK) return none();
  Py_RETURN_TRUE;
}

// (k_pool, v_pool, block_ids, head_dim, dtype code, lengths or None, fill_past) -> (key, value)
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 7) return none();
  const int dev = c10::cuda::current_device();
  const Tensor* ids = longs(a[2], dev, 2);
  const Tensor* lens = a[5] == Py_None ? nullptr : longs(a[5], dev, 1);
  const long d = PyLong_AsLong(a[3]), code = PyLong_AsLong(a[4]);
  const int fill = PyObject_IsTrue(a[6]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  Pools p;
  if (!ids || (a[5] != Py_None && (!lens || lens->size(0) != ids->size(0))) || !pools_of(a[0], a[1], d, dev, p)) return none();
  const at::ScalarType type = code == MI_F32 ? at::kFloat : code == MI_BF16 ? at::kBFloat16 : at::kHalf;
  const int64_t b = ids->size(0), nb = ids->size(1);
  const auto options = at::TensorOptions().dtype(type).device(p.k->device());
  const std::vector<int64_t> shape = {b, nb, p.bs, p.h, d};
  Tensor key = at::empty(shape, options), value = at::empty(shape, options);
  const int rc = mi_kv4_gather_blocks(p.k->data_ptr(), p.v->data_ptr(), static_cast<const int64_t*>(ids->data_ptr()), nb,
                                      lens ? static_cast<const int64_t*>(lens->data_ptr()) : nullptr, fill, b, nb,
                                      key.data_ptr(), value.data_ptr(), p.n, p.bs, (int)p.h, (int)d, (int)code,
                                      stream_of(dev));
  if (rc != MI_OK) return none();
  PyObject* k = THPVariable_Wrap(std::move(key));
  PyObject* v = THPVariable_Wrap(std::move(value));
  PyObject* both = k && v ? PyTuple_Pack(2, k, v) : nullptr;
  Py_XDECREF(k);
  Py_XDECREF(v);
  return both;
}

// (pools, pairs) -> True: a list or tuple of contiguous [num_blocks, ...] tensors of the same blocks and bytes
PyObject* copy_blocks(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (n_args != 2 || !(PyList_CheckExact(a[0]) || PyTuple_CheckExact(a[0]))) return none();
  const int dev = c10::cuda::current_device();
  const Tensor* pairs = longs(a[1], dev, 2);
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[0]);
  if (!pairs || pairs->size(1) != 2 || count < 1 || count > (1 << 20)) return none();
  std::vector<void*> table((size_t)count);
  int64_t blocks = 0, bytes = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor* t = plain(PySequence_Fast_GET_ITEM(a[0], i), dev);
    if (!t || t->dim() < 2 || !t->is_contiguous()) return none();
    if (i == 0) {
      blocks = t->size(0);
      bytes = (int64_t)t->nbytes();
    }
    if (t->size(0) != blocks || (int64_t)t->nbytes() != bytes) return none();
    table[(size_t)i] = t->data_ptr();
  }
  if (blocks < 1 || bytes < 1) return none();
  const int rc = mi_kv_copy_blocks(table.data(), (int)count, static_cast<const int64_t*>(pairs->data_ptr()), pairs->size(0),
                                   blocks, bytes / blocks, stream_of(dev));
  if (rc != MI_OK) return none();
  Py_RETURN_TRUE;
}

// No C++ exception (an allocation that fails) leaves a call: it becomes the ordinary path's error.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

#define MI_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<fn>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    MI_METHOD("kv4_paged_decode", decode), MI_METHOD("kv4_append", append), MI_METHOD("kv4_store_chunks", store_chunks),
    MI_METHOD("kv4_gather_blocks", gather), MI_METHOD("kv_copy_blocks", copy_blocks), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mi_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mi_calls() { return PyModule_Create(&module); }
