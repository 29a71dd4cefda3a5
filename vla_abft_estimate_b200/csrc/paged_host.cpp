// paged_host.cpp - the short way from Python to the paged cache's entry points.
//
// A paged call is a few microseconds of GPU time for small batches, and the
// Python checks, ctypes and allocations around it cost more than that. This
// extension takes a call whose arguments are all in order (types, shapes,
// strides, alignment, device) straight to the C ABI: about 5 us instead of 10.
// (Calls: one layer's cache; Layers: what is done for all layers of a model.)
// Anything else returns None, and vla_abft_estimate_b200/paged.py handles it:
// copies what has to be copied, refuses what is wrong and says why.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/EmptyTensor.h>
#include <ATen/TracerMode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
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
typedef int (*AppendAtFn)(const abft_kv_append_at_args*, void*);
typedef int (*TreeFn)(const abft_paged_tree_args*, void*);
typedef size_t (*TreeBytesFn)(const abft_paged_tree_args*);
typedef int (*AcceptFn)(const abft_draft_accept_args*, void*);
typedef int (*KeepFn)(const abft_kv_keep_args*, void*);
typedef int (*ForkFn)(const abft_kv_fork_args*, void*);

struct Calls {
  PyObject_HEAD
  abft_paged_kv kv;
  int device;
  AppendFn append;
  AttnFn attend[2];    // decode, prefill
  BytesFn scratch[2];
  PyObject* pages[2];  // the tensors behind kv, or NULL
  AppendAtFn append_at;
  TreeFn tree;
  TreeBytesFn tree_scratch;
};

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

at::ScalarType type_of(const Calls* c) { return c->kv.dtype == ABFT_DTYPE_F16 ? at::kHalf : at::kBFloat16; }

bool differentiated(const at::Tensor* t) { return t->requires_grad() && c10::GradMode::is_enabled(); }

// Nothing is traced, and no level of forward mode is open, in which any tensor
// may be a dual.
bool plain_mode() {
  return !at::tracer::impl::is_dispatch_enabled() && torch::autograd::ForwardADLevel::try_get_by_idx(0) == nullptr;
}

// The cache is known and asks for no gradient.
bool ready(const Calls* c) {
  return c->append != nullptr && c10::cuda::current_device() == c->device && c->pages[0] != nullptr && plain_mode() &&
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

// `size` whole numbers one after another (any number when it is negative).
bool list_of(int device, const at::Tensor* t, int64_t size, at::ScalarType type) {
  return t != nullptr && t->is_cuda() && t->get_device() == device && t->scalar_type() == type && t->dim() == 1 &&
         (size < 0 || t->size(0) == size) && (t->size(0) <= 1 || t->stride(0) == 1);
}

bool boundaries(const Calls* c, const at::Tensor* t) { return list_of(c->device, t, c->kv.batch + 1, at::kInt); }

bool group(const Calls* c, int64_t heads) {
  return heads > 0 && heads % c->kv.kv_heads == 0 && heads / c->kv.kv_heads <= 64;
}

void* stream_of(const Calls* c) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(c->device)).stream(); }

at::Tensor fresh(const Calls* c, at::IntArrayRef size, at::ScalarType type) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::kCUDA, static_cast<c10::DeviceIndex>(c->device)));
}

// append(q, k, v, rope or None, cu_seqlens or None, q_out or None, and, by
// positions of the caller's, positions and a tuple of sections): the rotated q;
// None when the call needs the long way; a status code.
PyObject* calls_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Calls* c = reinterpret_cast<const Calls*>(self);
  if ((n != 6 && n != 8) || !ready(c) || (n == 8 && c->append_at == nullptr)) Py_RETURN_NONE;
  const at::Tensor *q = tensor_of(a[0]), *k = tensor_of(a[1]), *v = tensor_of(a[2]);
  const at::Tensor *rope = tensor_of(a[3]), *cu = tensor_of(a[4]), *out = tensor_of(a[5]);
  if (!rows(c, k, -1, c->kv.kv_heads)) Py_RETURN_NONE;
  const int64_t tokens = k->size(0);
  if (!rows(c, v, tokens, c->kv.kv_heads) || !rows(c, q, tokens, -1) || !group(c, q->size(1))) Py_RETURN_NONE;
  abft_kv_append_at_args by;
  memset(&by, 0, sizeof by);
  abft_kv_append_args& args = by.append;
  if (n == 8) {
    const at::Tensor* at = tensor_of(a[6]);
    if (a[3] == Py_None || at == nullptr || !at->is_cuda() || at->get_device() != c->device || at->scalar_type() != at::kInt ||
        at->dim() != 2 || at->size(1) != tokens || (tokens > 1 && at->stride(1) != 1) || at->stride(0) < 0 ||
        !PyTuple_CheckExact(a[7]) || PyTuple_GET_SIZE(a[7]) != at->size(0) || at->size(0) < 1 || at->size(0) > ABFT_MOST_AXES)
      Py_RETURN_NONE;
    by.axes = static_cast<int32_t>(at->size(0));
    int64_t all = 0;
    for (int i = 0; i < by.axes; ++i) {
      PyObject* x = PyTuple_GET_ITEM(a[7], i);
      const long pairs = PyLong_CheckExact(x) ? PyLong_AsLong(x) : -1;
      if (pairs < 0 || pairs > INT32_MAX) {
        PyErr_Clear();
        Py_RETURN_NONE;
      }
      by.sections[i] = static_cast<int32_t>(pairs);
      all += pairs;
    }
    if (all * 2 != c->kv.head_dim) Py_RETURN_NONE;
    by.positions = static_cast<const int32_t*>(at->const_data_ptr());
    by.position_stride = at->stride(0);
  }
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
  Py_BEGIN_ALLOW_THREADS rc = n == 8 ? c->append_at(&by, stream) : c->append(&args, stream);
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

// Attention: decode (which 0), prefill (1) or a tree's (2, with parents).
PyObject* attend(const Calls* c, int which, PyObject* q_, PyObject* cu_, PyObject* parents_, PyObject* scale_, PyObject* out_,
                 PyObject* splits_, PyObject* sms_) {
  const at::Tensor *q = tensor_of(q_), *cu = tensor_of(cu_), *out = tensor_of(out_);
  if (!rows(c, q, which == 0 ? c->kv.batch : -1, -1) || !group(c, q->size(1))) Py_RETURN_NONE;
  abft_paged_tree_args tree;
  memset(&tree, 0, sizeof tree);
  abft_paged_attn_args& args = tree.attn;
  if (which != 0) {
    if (!boundaries(c, cu)) Py_RETURN_NONE;
    args.cu_seqlens = static_cast<const int32_t*>(cu->const_data_ptr());
  }
  if (which == 2) {
    const at::Tensor* parents = tensor_of(parents_);
    if (c->tree == nullptr || repeats(q) || !list_of(c->device, parents, q->size(0), at::kInt)) Py_RETURN_NONE;
    tree.parents = static_cast<const int32_t*>(parents->const_data_ptr());
  }
  double scale = 1.0 / sqrt(static_cast<double>(c->kv.head_dim));
  if (scale_ != Py_None) {
    if (!PyFloat_CheckExact(scale_)) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(scale_);
  }
  args.scale = static_cast<float>(scale);
  if (!PyLong_CheckExact(splits_) || !PyLong_CheckExact(sms_)) Py_RETURN_NONE;
  const long splits = PyLong_AsLong(splits_), sms = PyLong_AsLong(sms_);
  if (PyErr_Occurred() != nullptr || splits < 0 || sms < 0 || splits > INT32_MAX || sms > INT32_MAX ||
      !std::isfinite(args.scale)) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  args.num_splits = static_cast<int32_t>(splits);
  args.num_sms = static_cast<int32_t>(sms);
  at::Tensor made, space;
  if (out_ != Py_None) {
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
  const size_t need = which == 2 ? c->tree_scratch(&tree) : c->scratch[which](&args);
  if (need > 0) {
    // Of this call alone: calls of other threads or graphs have their own.
    space = fresh(c, {static_cast<int64_t>(need)}, at::kByte);
    args.workspace = space.data_ptr();
    args.workspace_bytes = need;
  }
  void* stream = stream_of(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = which == 2 ? c->tree(&tree, stream) : c->attend[which](&args, stream);
  Py_END_ALLOW_THREADS if (rc != ABFT_OK) return PyLong_FromLong(rc);
  if (out_ != Py_None) {
    written(*out);
    Py_INCREF(out_);
    return out_;
  }
  return THPVariable_Wrap(std::move(made));
}

// attend(prefill, q, cu_seqlens or None, scale or None, out or None,
// num_splits, num_sms): the output; None; a status code.
PyObject* calls_attend(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Calls* c = reinterpret_cast<const Calls*>(self);
  if (n != 7 || !ready(c)) Py_RETURN_NONE;
  return attend(c, a[0] == Py_True ? 1 : 0, a[1], a[2], Py_None, a[3], a[4], a[5], a[6]);
}

// tree(q, cu_seqlens, parents, scale or None, out or None, num_splits, num_sms):
// the same.
PyObject* calls_tree(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Calls* c = reinterpret_cast<const Calls*>(self);
  if (n != 7 || !ready(c)) Py_RETURN_NONE;
  return attend(c, 2, a[0], a[1], a[2], a[3], a[4], a[5], a[6]);
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

// drafts(addresses of append by positions, tree attention, its scratch size).
PyObject* calls_drafts(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  Calls* c = reinterpret_cast<Calls*>(self);
  unsigned long long fn[3] = {0, 0, 0};
  for (int i = 0; i < 3 && n == 3; ++i) {
    fn[i] = PyLong_AsUnsignedLongLong(a[i]);
    if (PyErr_Occurred() != nullptr) return nullptr;
  }
  if (n != 3) {
    PyErr_SetString(PyExc_TypeError, "drafts takes three addresses");
    return nullptr;
  }
  c->append_at = reinterpret_cast<AppendAtFn>(fn[0]);
  c->tree = reinterpret_cast<TreeFn>(fn[1]);
  c->tree_scratch = reinterpret_cast<TreeBytesFn>(fn[2]);
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
    {"tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_tree>)), METH_FASTCALL, nullptr},
    {"drafts", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_drafts>)), METH_FASTCALL, nullptr},
    {"hold", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<calls_hold>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyTypeObject calls_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

// ---- a model's layers -------------------------------------------------------------
struct Layers {
  PyObject_HEAD
  abft_paged_kv kv;
  int device;
  int32_t layers;
  PyObject* pools;   // bytes: the pools' addresses
  AcceptFn accept;
  KeepFn keep;
  ForkFn fork;
  PyObject* pages;   // tuple of every layer's page tensors
  PyObject* table;
  PyObject* lens;
};

bool layers_ready(const Layers* c) {
  if (c->accept == nullptr || c->pages == nullptr || c10::cuda::current_device() != c->device || !plain_mode()) return false;
  if (c10::GradMode::is_enabled())
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(c->pages); ++i)
      if (THPVariable_Unpack(PyTuple_GET_ITEM(c->pages, i)).requires_grad()) return false;
  return true;
}

void pages_written(const Layers* c) {
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(c->pages); ++i) written(THPVariable_Unpack(PyTuple_GET_ITEM(c->pages, i)));
}

void* layers_stream(const Layers* c) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(c->device)).stream();
}

const int32_t* int_ptr(const at::Tensor* t) { return static_cast<const int32_t*>(t->const_data_ptr()); }

// accept(cu_seqlens, parents, ids, answers): (kept, counts, next); None; a status
// code.
PyObject* layers_accept(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Layers* c = reinterpret_cast<const Layers*>(self);
  if (n != 4 || c->accept == nullptr || c10::cuda::current_device() != c->device || !plain_mode()) Py_RETURN_NONE;
  const at::Tensor *cu = tensor_of(a[0]), *parents = tensor_of(a[1]), *ids = tensor_of(a[2]), *answers = tensor_of(a[3]);
  if (ids == nullptr || (ids->scalar_type() != at::kLong && ids->scalar_type() != at::kInt)) Py_RETURN_NONE;
  const at::ScalarType type = ids->scalar_type();
  if (!list_of(c->device, ids, -1, type) || !list_of(c->device, answers, ids->size(0), type) ||
      !list_of(c->device, parents, ids->size(0), at::kInt) || !list_of(c->device, cu, c->kv.batch + 1, at::kInt))
    Py_RETURN_NONE;
  // A memory of its own for each, which the caller may resize, hand to a stream or free;
  // asked for on the current device, which is the layers', without a dispatcher's way each.
  auto list = [](int64_t size, at::ScalarType type) {
    return at::Tensor(at::detail::empty_generic({size}, c10::cuda::CUDACachingAllocator::get(),
                                                c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
  };
  at::Tensor kept = list(ids->size(0), at::kInt), counts = list(c->kv.batch, at::kInt), next = list(c->kv.batch, type);
  abft_draft_accept_args args;
  memset(&args, 0, sizeof args);
  args.cu_seqlens = int_ptr(cu), args.parents = int_ptr(parents);
  args.ids = ids->const_data_ptr(), args.answers = answers->const_data_ptr();
  args.kept = static_cast<int32_t*>(kept.data_ptr());
  args.counts = static_cast<int32_t*>(counts.data_ptr());
  args.next = next.data_ptr();
  args.status = c->kv.status;
  args.tokens = ids->size(0);
  args.batch = c->kv.batch;
  args.id_bytes = type == at::kLong ? 8 : 4;
  void* stream = layers_stream(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = c->accept(&args, stream);
  Py_END_ALLOW_THREADS if (rc != ABFT_OK) return PyLong_FromLong(rc);
  PyObject* x = THPVariable_Wrap(std::move(kept));
  PyObject* y = THPVariable_Wrap(std::move(counts));
  PyObject* z = THPVariable_Wrap(std::move(next));
  PyObject* all = x != nullptr && y != nullptr && z != nullptr ? PyTuple_Pack(3, x, y, z) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  Py_XDECREF(z);
  return all;
}

// keep(cu_seqlens, kept, counts, lens_out): a status code; None.
PyObject* layers_keep(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Layers* c = reinterpret_cast<const Layers*>(self);
  if (n != 4 || !layers_ready(c)) Py_RETURN_NONE;
  const at::Tensor *cu = tensor_of(a[0]), *kept = tensor_of(a[1]), *counts = tensor_of(a[2]), *out = tensor_of(a[3]);
  if (!list_of(c->device, cu, c->kv.batch + 1, at::kInt) || !list_of(c->device, kept, -1, at::kInt) ||
      !list_of(c->device, counts, c->kv.batch, at::kInt) || !list_of(c->device, out, c->kv.batch, at::kInt))
    Py_RETURN_NONE;
  abft_kv_keep_args args;
  memset(&args, 0, sizeof args);
  args.kv = c->kv;
  args.pools = reinterpret_cast<void* const*>(PyBytes_AS_STRING(c->pools));
  args.layers = c->layers;
  args.cu_seqlens = int_ptr(cu), args.kept = int_ptr(kept), args.counts = int_ptr(counts);
  args.lens_out = static_cast<int32_t*>(out->data_ptr());
  args.tokens = kept->size(0);
  void* stream = layers_stream(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = c->keep(&args, stream);
  Py_END_ALLOW_THREADS if (rc == ABFT_OK) {
    pages_written(c);
    written(*out);
  }
  return PyLong_FromLong(rc);
}

// fork(src, dst, pages): a status code; None.
PyObject* layers_fork(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  const Layers* c = reinterpret_cast<const Layers*>(self);
  if (n != 3 || !layers_ready(c)) Py_RETURN_NONE;
  const at::Tensor *src = tensor_of(a[0]), *dst = tensor_of(a[1]), *pages = tensor_of(a[2]);
  if (!list_of(c->device, src, -1, at::kInt) || src->size(0) > INT32_MAX || !list_of(c->device, dst, src->size(0), at::kInt) ||
      !list_of(c->device, pages, src->size(0), at::kInt))
    Py_RETURN_NONE;
  abft_kv_fork_args args;
  memset(&args, 0, sizeof args);
  args.kv = c->kv;
  args.pools = reinterpret_cast<void* const*>(PyBytes_AS_STRING(c->pools));
  args.layers = c->layers;
  args.src = int_ptr(src), args.dst = int_ptr(dst), args.pages = int_ptr(pages);
  args.pairs = static_cast<int32_t>(src->size(0));
  void* stream = layers_stream(c);
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = c->fork(&args, stream);
  Py_END_ALLOW_THREADS if (rc == ABFT_OK) {
    pages_written(c);
    written(THPVariable_Unpack(c->table));
    written(THPVariable_Unpack(c->lens));
  }
  return PyLong_FromLong(rc);
}

void layers_dealloc(PyObject* self) {
  Layers* c = reinterpret_cast<Layers*>(self);
  Py_CLEAR(c->pools);
  Py_CLEAR(c->pages);
  Py_CLEAR(c->table);
  Py_CLEAR(c->lens);
  Py_TYPE(self)->tp_free(self);
}

// Layers(kv bytes, device, bytes of the pools' addresses, addresses of accept, keep,
// fork, tuple of page tensors, page table, lengths).
int layers_init(PyObject* self, PyObject* args, PyObject*) {
  Layers* c = reinterpret_cast<Layers*>(self);
  const char* kv;
  Py_ssize_t size;
  unsigned long long fn[3];
  PyObject *pools, *pages, *table, *lens;
  if (!PyArg_ParseTuple(args, "y#iO!KKKO!OO", &kv, &size, &c->device, &PyBytes_Type, &pools, fn, fn + 1, fn + 2, &PyTuple_Type,
                        &pages, &table, &lens))
    return -1;
  bool tensors = THPVariable_Check(table) && THPVariable_Check(lens);
  tensors = tensors && PyBytes_GET_SIZE(pools) == static_cast<Py_ssize_t>(sizeof(void*)) * PyTuple_GET_SIZE(pages);
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(pages); ++i) tensors = tensors && THPVariable_Check(PyTuple_GET_ITEM(pages, i));
  if (size != static_cast<Py_ssize_t>(sizeof c->kv) || !tensors) {
    PyErr_SetString(PyExc_ValueError, "the cache struct has another size, or no tensors follow");
    return -1;
  }
  memcpy(&c->kv, kv, sizeof c->kv);
  c->layers = static_cast<int32_t>(PyTuple_GET_SIZE(pages) / 2);
  Py_INCREF(pools);
  Py_XSETREF(c->pools, pools);
  Py_INCREF(pages);
  Py_XSETREF(c->pages, pages);
  Py_INCREF(table);
  Py_XSETREF(c->table, table);
  Py_INCREF(lens);
  Py_XSETREF(c->lens, lens);
  c->accept = reinterpret_cast<AcceptFn>(fn[0]);
  c->keep = reinterpret_cast<KeepFn>(fn[1]);
  c->fork = reinterpret_cast<ForkFn>(fn[2]);
  return 0;
}

PyMethodDef layers_methods[] = {
    {"accept", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<layers_accept>)), METH_FASTCALL, nullptr},
    {"keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<layers_keep>)), METH_FASTCALL, nullptr},
    {"fork", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<layers_fork>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyTypeObject layers_type = {PyVarObject_HEAD_INIT(nullptr, 0)};

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
  layers_type.tp_name = "_paged_host.Layers";
  layers_type.tp_basicsize = sizeof(Layers);
  layers_type.tp_flags = Py_TPFLAGS_DEFAULT;
  layers_type.tp_new = PyType_GenericNew;
  layers_type.tp_init = layers_init;
  layers_type.tp_dealloc = layers_dealloc;
  layers_type.tp_methods = layers_methods;
  if (PyType_Ready(&calls_type) < 0 || PyType_Ready(&layers_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module_def);
  if (m == nullptr) return nullptr;
  Py_INCREF(&calls_type);
  if (PyModule_AddObject(m, "Calls", reinterpret_cast<PyObject*>(&calls_type)) < 0) {
    Py_DECREF(&calls_type);
    Py_DECREF(m);
    return nullptr;
  }
  Py_INCREF(&layers_type);
  if (PyModule_AddObject(m, "Layers", reinterpret_cast<PyObject*>(&layers_type)) < 0) {
    Py_DECREF(&layers_type);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
