// paged_host.cpp - the short way from Python to the paged cache's entry points.
//
// A paged call is a few microseconds of GPU time for small batches, and the
// Python checks, ctypes and allocations around it cost more than that. This
// extension takes a call whose arguments are all in order (types, shapes,
// strides, alignment, device) straight to the C ABI: about 5 us instead of 10.
// Anything else returns None, and vla_abft_estimate_b200/paged.py handles it:
// copies what has to be copied, refuses what is wrong and says why.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <math.h>
#include <string.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/abft_b200.h"

namespace {

typedef int (*AppendFn)(const abft_kv_append_args*, void*);
typedef int (*AttnFn)(const abft_paged_attn_args*, void*);
typedef size_t (*BytesFn)(const abft_paged_attn_args*);

struct Calls {
  PyObject_HEAD
  abft_paged_kv kv;
  int device;
  AppendFn append;
  AttnFn attend[2];    // decode, prefill
  BytesFn scratch[2];
  PyObject* pages[2];  // the tensors behind kv, or NULL
};

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

at::ScalarType type_of(const Calls* c) { return c->kv.dtype == ABFT_DTYPE_F16 ? at::kHalf : at::kBFloat16; }

bool differentiated(const at::Tensor* t) { return t->requires_grad() && c10::GradMode::is_enabled(); }

// The cache is known and asks for no gradient; nothing is traced, and no level
// of forward mode is open, in which any tensor may be a dual.
bool ready(const Calls* c) {
  return c->append != nullptr && c10::cuda::current_device() == c->device && c->pages[0] != nullptr &&
         !at::tracer::impl::is_dispatch_enabled() && torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr &&
         !differentiated(&THPVariable_Unpack(c->pages[0])) && !differentiated(&THPVariable_Unpack(c->pages[1]));
}

// Autograd learns that the tensor has been written.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// [tokens, heads, head_dim] rows the kernels can read or write in place.
bool rows(const Calls* c, const at::Tensor* t, int64_t tokens, int64_t heads) {
  if (t == nullptr || !t->is_cuda() || t->get_device() != c->device || t->scalar_type() != type_of(c) || t->dim() != 3)
    return false;
  const auto size = t->sizes();
  const auto stride = t->strides();
  return size[2] == c->kv.head_dim && (tokens < 0 || size[0] == tokens) && (heads < 0 || size[1] == heads) &&
         stride[2] == 1 && stride[0] % 8 == 0 && stride[1] % 8 == 0 &&
         (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15u) == 0 && !differentiated(t);
}

bool repeats(const at::Tensor* t) {
  return (t->stride(0) == 0 && t->size(0) > 1) || (t->stride(1) == 0 && t->size(1) > 1);
}

bool boundaries(const Calls* c, const at::Tensor* t) {
  return t != nullptr && t->is_cuda() && t->get_device() == c->device && t->scalar_type() == at::kInt && t->dim() == 1 &&
         t->size(0) == c->kv.batch + 1 && (t->size(0) == 1 || t->stride(0) == 1);
}

bool group(const Calls* c, int64_t heads) {
  return heads > 0 && heads % c->kv.kv_heads == 0 && heads / c->kv.kv_heads <= 64;
}

void* stream_of(const Calls* c) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(c->device)).stream(); }

at::Tensor fresh(const Calls* c, at::IntArrayRef size, at::ScalarType type) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(c->device)));
}

// append(q, k, v, rope or None, cu_seqlens or None, q_out or None): the
// rotated q; None when the call needs the long way; a status code.
PyObject* calls_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Calls* c = reinterpret_cast<const Calls*>(self);
  if (n != 6 || !ready(c)) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]);
  const at::Tensor *rope = tensor_of(a[3]), *cu = tensor_of(a[4]), *out = tensor_of(a[5]);
  if (!rows(c, k, -1, c->kv.kv_heads)) Py_RETURN_NONE;
  const int64_t tokens = k->size(0);
  if (!rows(c, v, tokens, c->kv.kv_heads) || !rows(c, q, tokens, -1) || !group(c, q->size(1))) Py_RETURN_NONE;
  abft_kv_append_args args;
  memset(&args, 0, sizeof args);
  if (a[3] != Py_None) {
    if (rope == nullptr || !rope->is_cuda() || rope->get_device() != c->device || rope->scalar_type() != at::kFloat ||
        rope->dim() != 3 || rope->size(0) == 0 || rope->size(1) * 2 != c->kv.head_dim || rope->size(2) != 2 ||
        !rope->is_contiguous() || differentiated(rope) || (reinterpret_cast<uintptr_t>(rope->const_data_ptr()) & 15u) != 0)
      Py_RETURN_NONE;
    args.rope = static_cast<const float*>(rope->const_data_ptr());
    args.max_positions = rope->size(0);
  }
  if (a[4] != Py_None) {
    if (!boundaries(c, cu)) Py_RETURN_NONE;
    args.cu_seqlens = static_cast<const int32_t*>(cu->const_data_ptr());
  } else if (tokens != c->kv.batch) {
    Py_RETURN_NONE;
  }
  at::Tensor made;
  if (a[5] != Py_None) {
    if (!rows(c, out, tokens, q->size(1)) || repeats(out)) Py_RETURN_NONE;
  } else {
    made = fresh(c, q->sizes(), type_of(c));
    out = &made;
  }
  args.kv = c->kv;
  args.q = q->const_data_ptr(), args.k = k->const_data_ptr(), args.v = v->const_data_ptr();
  args.q_out = out->data_ptr();
  args.q_token_stride = q->stride(0), args.q_head_stride = q->stride(1);
  args.k_token_stride = k->stride(0), args.k_head_stride = k->stride(1);
  args.v_token_stride = v->stride(0), args.v_head_stride = v->stride(1);
  args.o_token_stride = out->stride(0), args.o_head_stride = out->stride(1);
  args.tokens = tokens;
  args.heads = static_cast<int32_t>(q->size(1));
  void* stream = stream_of(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = c->append(&args, stream);
  Py_END_ALLOW_THREADS if (rc != ABFT_OK) return PyLong_FromLong(rc);
  written(THPVariable_Unpack(c->pages[0]));
  written(THPVariable_Unpack(c->pages[1]));
  if (a[5] != Py_None) {
    written(*out);
    Py_INCREF(a[5]);
    return a[5];
  }
  return THPVariable_Wrap(std::move(made));
}

// attend(prefill, q, cu_seqlens or None, scale or None, out or None,
// num_splits, num_sms): the output; None; a status code.
PyObject* calls_attend(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Calls* c = reinterpret_cast<const Calls*>(self);
  if (n != 7 || !ready(c)) Py_RETURN_NONE;
  const int which = a[0] == Py_True ? 1 : 0;
  const at::Tensor *q = tensor_of(a[1]), *cu = tensor_of(a[2]), *out = tensor_of(a[4]);
  if (!rows(c, q, which == 0 ? c->kv.batch : -1, -1) || !group(c, q->size(1))) Py_RETURN_NONE;
  abft_paged_attn_args args;
  memset(&args, 0, sizeof args);
  if (which == 1) {
    if (!boundaries(c, cu)) Py_RETURN_NONE;
    args.cu_seqlens = static_cast<const int32_t*>(cu->const_data_ptr());
  }
  double scale = 1.0 / sqrt(static_cast<double>(c->kv.head_dim));
  if (a[3] != Py_None) {
    if (!PyFloat_CheckExact(a[3])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(a[3]);
  }
  args.scale = static_cast<float>(scale);
  if (!PyLong_CheckExact(a[5]) || !PyLong_CheckExact(a[6])) Py_RETURN_NONE;
  const long splits = PyLong_AsLong(a[5]), sms = PyLong_AsLong(a[6]);
  if (PyErr_Occurred() != nullptr || splits < 0 || sms < 0 || splits > INT32_MAX || sms > INT32_MAX ||
      !std::isfinite(args.scale)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  args.num_splits = static_cast<int32_t>(splits);
  args.num_sms = static_cast<int32_t>(sms);
  at::Tensor made, space;
  if (a[4] != Py_None) {
    if (!rows(c, out, q->size(0), q->size(1)) || repeats(out)) Py_RETURN_NONE;
  } else {
    made = fresh(c, q->sizes(), type_of(c));
    out = &made;
  }
  args.kv = c->kv;
  args.q = q->const_data_ptr();
  args.out = out->data_ptr();
  args.q_token_stride = q->stride(0), args.q_head_stride = q->stride(1);
  args.o_token_stride = out->stride(0), args.o_head_stride = out->stride(1);
  args.tokens = q->size(0);
  args.heads = static_cast<int32_t>(q->size(1));
  const size_t need = c->scratch[which](&args);
  if (need > 0) {
    // Of this call alone: calls of other threads or graphs have their own.
    space = fresh(c, {static_cast<int64_t>(need)}, at::kByte);
    args.workspace = space.data_ptr();
    args.workspace_bytes = need;
  }
  void* stream = stream_of(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = c->attend[which](&args, stream);
  Py_END_ALLOW_THREADS if (rc != ABFT_OK) return PyLong_FromLong(rc);
  if (a[4] != Py_None) {
    written(*out);
    Py_INCREF(a[4]);
    return a[4];
  }
  return THPVariable_Wrap(std::move(made));
}

// An exception of torch's (out of memory, say) becomes a Python one.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type != nullptr) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// hold(k_pages, v_pages): the tensors whose addresses the cache struct has.
PyObject* calls_hold(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Calls* c = reinterpret_cast<Calls*>(self);
  if (n != 2 || !THPVariable_Check(a[0]) || !THPVariable_Check(a[1])) {
    PyErr_SetString(PyExc_TypeError, "hold takes the two page tensors");
    return nullptr;
  }
  for (int i = 0; i < 2; ++i) {
    Py_INCREF(a[i]);
    Py_XSETREF(c->pages[i], a[i]);
  }
  Py_RETURN_NONE;
}

void calls_dealloc(PyObject* self) {
  Calls* c = reinterpret_cast<Calls*>(self);
  Py_CLEAR(c->pages[0]);
  Py_CLEAR(c->pages[1]);
  Py_TYPE(self)->tp_free(self);
}

// Calls(kv bytes, device, addresses of append, decode, its scratch size,
// prefill, its scratch size).
int calls_init(PyObject* self, PyObject* args, PyObject*) {
  Calls* c = reinterpret_cast<Calls*>(self);
  const char* kv;
  Py_ssize_t size;
  unsigned long long fn[5];
  if (!PyArg_ParseTuple(args, "y#iKKKKK", &kv, &size, &c->device, fn, fn + 1, fn + 2, fn + 3, fn + 4)) return -1;
  if (size != static_cast<Py_ssize_t>(sizeof c->kv)) {
    PyErr_SetString(PyExc_ValueError, "the cache struct has another size");
    return -1;
  }
  memcpy(&c->kv, kv, sizeof c->kv);
  c->append = reinterpret_cast<AppendFn>(fn[0]);
  c->attend[0] = reinterpret_cast<AttnFn>(fn[1]);
  c->scratch[0] = reinterpret_cast<BytesFn>(fn[2]);
  c->attend[1] = reinterpret_cast<AttnFn>(fn[3]);
  c->scratch[1] = reinterpret_cast<BytesFn>(fn[4]);
  return 0;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_append>)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_attend>)), METH_FASTCALL, nullptr},
    {"hold", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_hold>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyTypeObject calls_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_host(void) {
  calls_type.tp_name = "_paged_host.Calls";
  calls_type.tp_basicsize = sizeof(Calls);
  calls_type.tp_flags = Py_TPFLAGS_DEFAULT;
  calls_type.tp_new = PyType_GenericNew;
  calls_type.tp_init = calls_init;
  calls_type.tp_dealloc = calls_dealloc;
  calls_type.tp_methods = methods;
  if (PyType_Ready(&calls_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (m == nullptr) return nullptr;
  Py_INCREF(&calls_type);
  if (PyModule_AddObject(m, "Calls", reinterpret_cast<PyObject*>(&calls_type)) < 0) {
    Py_DECREF(&calls_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
