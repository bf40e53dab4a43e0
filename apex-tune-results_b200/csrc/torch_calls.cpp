// The short way from Python to the paged cache operators: checks, allocation and the C call in
// C++, for well-formed arguments. Each function returns None for anything else (another
// layout, type or device, a tensor subclass, a failing call); apex_attn/paged.py then takes its own way,
// which copies what can be copied and raises what has to be raised. Both make the same calls of
// the C ABI, whose addresses `init` gets, so this file links to nothing of the library.
//
// Measured on the host of a B200, Python alone / this: attention 15.9 / 7.4 us per call, append 8.0 /
// 3.4 us, plan and release together 24 / 11 us; the kernels of a small decode step take as long.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <Python.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <exception>

#include "apex_attn.h"

namespace {

struct Calls {
  decltype(&apex_attn_kv_plan) plan = nullptr;
  decltype(&apex_attn_kv_release) release = nullptr;
  decltype(&apex_attn_kv_append) append = nullptr;
  decltype(&apex_attn_fwd_paged_workspace_bytes) workspace_bytes = nullptr;
  decltype(&apex_attn_fwd_paged) attend = nullptr;
} g;

// A plain CUDA tensor, or null. `device` is set by the first and has to be that of the others.
const at::Tensor* cuda_tensor(PyObject* o, int& device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) return nullptr;
  const int at = t.get_device();
  if (device < 0) device = at;
  return at == device ? &t : nullptr;
}

bool vector_of(const at::Tensor* t, at::ScalarType type, int64_t n) {
  return t != nullptr && t->scalar_type() == type && t->dim() == 1 && t->size(0) == n && t->is_contiguous();
}

uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

// [rows, H, D] with unit stride along D, the others multiples of 8, 16-byte aligned.
bool rows_ready(const at::Tensor& t) {
  return t.dim() == 3 && t.stride(2) == 1 && ((t.stride(0) | t.stride(1)) & 7) == 0 && t.stride(1) >= t.size(2) &&
         (address(t) & 15) == 0;
}

// Whether the (token, head) rows of an output do not overlap.
bool rows_distinct(const at::Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2), st = t.stride(0), sh = t.stride(1);
  return (n <= 1 || st >= d) && (h <= 1 || sh >= d) &&
         (n <= 1 || h <= 1 || st >= (h - 1) * sh + d || sh >= (n - 1) * st + d);
}

int dtype_of(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? APEX_ATTN_BF16 : t.scalar_type() == at::kHalf ? APEX_ATTN_FP16 : -1;
}

at::Tensor new_tensor(at::IntArrayRef size, at::ScalarType type, int device) {
  return at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (at::DeviceIndex)device), std::nullopt);
}

// `n` entries of a vector from `first` on, as a tensor of its own over the same storage. (Several small
// outputs share an allocation: one of their own each took about half a microsecond.)
at::Tensor part_of(const at::Tensor& t, int64_t first, int64_t n) {
  at::Tensor part = at::detail::make_tensor<at::TensorImpl>(at::TensorImpl::VIEW, c10::Storage(t.storage()),
                                                            t.key_set(), t.dtype());
  part.unsafeGetTensorImpl()->set_storage_offset(first);
  part.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return part;
}

// The cache of append and attend: pointers, sizes, and byte strides at strides[4 .. 9].
template <typename A>
bool cache_args(A& a, PyObject* const* o, int& device) {
  const at::Tensor* k = cuda_tensor(o[0], device);
  const at::Tensor* v = cuda_tensor(o[1], device);
  const at::Tensor* ks = cuda_tensor(o[2], device);
  const at::Tensor* vs = cuda_tensor(o[3], device);
  if (!k || !v || !ks || !vs || k->dim() != 4 || v->sizes() != k->sizes()) return false;
  const int64_t blocks = k->size(0), heads = k->size(1), block = k->size(2), dim = k->size(3);
  if (blocks <= 0 || blocks > INT_MAX || heads <= 0 || heads > INT_MAX || block > INT_MAX || dim > INT_MAX) return false;
  int i = 4;
  for (const at::Tensor* c : {k, v}) {
    if (c->scalar_type() != at::kFloat8_e4m3fn || c->stride(3) != 1) return false;
    const int64_t st = c->stride(2);
    const int64_t sh = heads > 1 ? c->stride(1) : block * dim, sb = blocks > 1 ? c->stride(0) : heads * block * dim;
    if (st < dim || ((sb | sh | st) & 15) != 0 || (address(*c) & 15) != 0) return false;
    a.strides[i++] = sb;
    a.strides[i++] = sh;
    a.strides[i++] = st;
  }
  for (const at::Tensor* s : {ks, vs})
    if (s->scalar_type() != at::kFloat || s->dim() != 2 || s->size(0) != blocks || s->size(1) != heads ||
        !s->is_contiguous())
      return false;
  a.k_cache = k->data_ptr();
  a.v_cache = v->data_ptr();
  a.k_scale = static_cast<float*>(ks->data_ptr());
  a.v_scale = static_cast<float*>(vs->data_ptr());
  a.num_blocks = (int)blocks;
  a.heads_kv = (int)heads;
  a.block_size = (int)block;
  a.head_dim = (int)dim;
  return true;
}

// A whole number that fits an int; false for None and anything else.
bool whole(PyObject* o, int& out) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow != 0 || v < INT_MIN || v > INT_MAX) return false;
  out = (int)v;
  return true;
}

// The block table: int32 [batch, width] with unit stride along its rows.
template <typename A>
bool table_args(A& a, const at::Tensor* t) {
  if (!t || t->scalar_type() != at::kInt || t->dim() != 2) return false;
  const int64_t batch = t->size(0), width = t->size(1);
  if (batch <= 0 || width <= 0 || batch > INT_MAX || width > INT_MAX) return false;
  if ((width > 1 && t->stride(1) != 1) || (batch > 1 && t->stride(0) < width)) return false;
  a.block_table = static_cast<int*>(t->data_ptr());
  a.batch = (int)batch;
  a.table_width = (int)width;
  a.table_stride = batch > 1 ? t->stride(0) : width;
  return true;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

template <typename F>
int without_gil(F&& call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS rc = call();
  Py_END_ALLOW_THREADS return rc;
}

// Runs a function body; a C++ exception (out of memory, say) is left to the other way to meet.
template <typename F>
PyObject* guarded(F&& body) {
  try {
    if (PyObject* result = body()) return result;
  } catch (const std::exception&) {
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// (q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens_q, max_seqlen_q, causal,
//  sm_scale, return_lse, window_left, out)
PyObject* attend(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 14 || !g.attend) return nullptr;
    apex_attn_paged_args a{};
    int device = -1;
    const at::Tensor* q = cuda_tensor(o[0], device);
    if (!q || !rows_ready(*q) || !cache_args(a, o + 1, device)) return nullptr;
    const int64_t total = q->size(0), heads = q->size(1);
    a.dtype = dtype_of(*q);
    if (a.dtype < 0 || total <= 0 || total > INT_MAX || heads <= 0 || heads > INT_MAX || q->size(2) != a.head_dim)
      return nullptr;
    if (!table_args(a, cuda_tensor(o[5], device))) return nullptr;
    const at::Tensor* lens = cuda_tensor(o[6], device);
    if (!vector_of(lens, at::kInt, a.batch)) return nullptr;
    int max_q = 0;
    if (o[7] == Py_None) {
      if (total % a.batch != 0) return nullptr;
      if (o[8] != Py_None && (!whole(o[8], max_q) || (int64_t)max_q * a.batch != total)) return nullptr;
      max_q = (int)(total / a.batch);
    } else {
      const at::Tensor* cu = cuda_tensor(o[7], device);
      if (!vector_of(cu, at::kInt, (int64_t)a.batch + 1) || !whole(o[8], max_q) || max_q < 1) return nullptr;
      a.cu_seqlens_q = static_cast<const int*>(cu->data_ptr());
      max_q = (int)std::min<int64_t>(max_q, total);
    }
    if ((o[9] != Py_True && o[9] != Py_False) || (o[11] != Py_True && o[11] != Py_False)) return nullptr;
    a.causal = o[9] == Py_True;
    a.sm_scale = (float)(1.0 / std::sqrt((double)a.head_dim));
    if (o[10] != Py_None) {
      if (!PyFloat_CheckExact(o[10])) return nullptr;
      a.sm_scale = (float)PyFloat_AS_DOUBLE(o[10]);
    }
    a.window_left = -1;
    if (o[12] != Py_None && (!whole(o[12], a.window_left) || a.window_left < 0 || !a.causal)) return nullptr;
    at::Tensor out;
    if (o[13] == Py_None) {
      out = new_tensor(q->sizes(), q->scalar_type(), device);
      a.zero_rest = 1;
    } else {
      const at::Tensor* given = cuda_tensor(o[13], device);
      if (!given || given->scalar_type() != q->scalar_type() || given->sizes() != q->sizes() || !rows_ready(*given) ||
          !rows_distinct(*given))
        return nullptr;
      out = *given;
    }
    at::Tensor lse;
    if (o[11] == Py_True) {
      // The kernel clears the rows outside every request, unless `out` keeps its own: the other way.
      if (a.zero_rest == 0 && a.cu_seqlens_q != nullptr) return nullptr;
      lse = new_tensor({heads, total}, at::kFloat, device);
      a.lse = static_cast<float*>(lse.data_ptr());
    }
    const size_t bytes = g.workspace_bytes((int)heads, a.heads_kv, max_q, a.head_dim);
    const at::Tensor workspace = new_tensor({(int64_t)bytes}, at::kByte, device);
    a.q = q->data_ptr();
    a.o = out.data_ptr();
    a.seq_lens = static_cast<const int*>(lens->data_ptr());
    a.strides[0] = q->stride(0);
    a.strides[1] = q->stride(1);
    a.strides[2] = out.stride(0);
    a.strides[3] = out.stride(1);
    a.heads_q = (int)heads;
    a.total_q = (int)total;
    a.max_seqlen_q = max_q;
    a.known_device = device + 1;
    void* stream = stream_of(device);
    if (without_gil([&] { return g.attend(&a, workspace.data_ptr(), bytes, stream); }) != APEX_ATTN_OK) return nullptr;
    PyObject* first = o[13] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(o[13]);
    if (first == nullptr || o[11] == Py_False) return first;
    PyObject* second = THPVariable_Wrap(lse);
    PyObject* both = second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_DECREF(first);
    Py_XDECREF(second);
    return both;
  });
}

// (k, v, k_cache, v_cache, k_scale, v_scale, slots): True when done
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 7 || !g.append) return nullptr;
    apex_attn_kv_append_args a{};
    int device = -1;
    const at::Tensor* k = cuda_tensor(o[0], device);
    const at::Tensor* v = cuda_tensor(o[1], device);
    if (!k || !v || !rows_ready(*k) || !rows_ready(*v) || k->sizes() != v->sizes() ||
        k->scalar_type() != v->scalar_type() || !cache_args(a, o + 2, device))
      return nullptr;
    const int64_t total = k->size(0);
    a.dtype = dtype_of(*k);
    if (a.dtype < 0 || total <= 0 || total > INT_MAX || k->size(1) != a.heads_kv || k->size(2) != a.head_dim)
      return nullptr;
    const at::Tensor* slots = cuda_tensor(o[6], device);
    if (!slots || slots->scalar_type() != at::kLong || slots->dim() != 1 || slots->size(0) < total ||
        !slots->is_contiguous())
      return nullptr;
    a.k = k->data_ptr();
    a.v = v->data_ptr();
    a.slots = reinterpret_cast<const long long*>(slots->data_ptr());
    a.total = (int)total;
    a.strides[0] = k->stride(0);
    a.strides[1] = k->stride(1);
    a.strides[2] = v->stride(0);
    a.strides[3] = v->stride(1);
    a.known_device = device + 1;
    void* stream = stream_of(device);
    if (without_gil([&] { return g.append(&a, stream); }) != APEX_ATTN_OK) return nullptr;
    Py_RETURN_TRUE;
  });
}

// What plan and release share: (block_table, seq_lens, new_lens or finished, free_blocks, free_count,
// block_size, ...)
bool bookkeeping_args(apex_attn_kv_plan_args& a, PyObject* const* o, bool plan, int& device) {
  if (!table_args(a, cuda_tensor(o[0], device))) return false;
  const at::Tensor* lens = cuda_tensor(o[1], device);
  const at::Tensor* third = cuda_tensor(o[2], device);
  const at::Tensor* blocks = cuda_tensor(o[3], device);
  const at::Tensor* count = cuda_tensor(o[4], device);
  if (!vector_of(lens, at::kInt, a.batch) || !vector_of(third, at::kInt, a.batch) || !blocks ||
      !vector_of(blocks, at::kInt, blocks->numel()) || blocks->numel() <= 0 || blocks->numel() > INT_MAX ||
      !vector_of(count, at::kInt, 1) || !whole(o[5], a.block_size))
    return false;
  a.seq_lens = static_cast<const int*>(lens->data_ptr());
  (plan ? a.new_lens : a.finished) = static_cast<const int*>(third->data_ptr());
  a.free_blocks = static_cast<int*>(blocks->data_ptr());
  a.free_count = static_cast<const int*>(count->data_ptr());
  a.free_capacity = (int)blocks->numel();
  a.known_device = device + 1;
  return true;
}

PyObject* wrapped(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) {
    PyObject* w = out ? THPVariable_Wrap(t) : nullptr;
    if (w == nullptr) {
      Py_XDECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, w);
  }
  return out;
}

// (..., max_new_tokens): (slots, cu_seqlens, seq_lens, free_count, placed)
PyObject* plan(PyObject*, PyObject* const* o, Py_ssize_t given) {
  return guarded([&]() -> PyObject* {
    if (given != 7 || !g.plan) return nullptr;
    apex_attn_kv_plan_args a{};
    int device = -1;
    if (!bookkeeping_args(a, o, true, device) || !whole(o[6], a.max_new_tokens) || a.max_new_tokens < 1) return nullptr;
    const at::Tensor slots = new_tensor({a.max_new_tokens}, at::kLong, device);
    const int64_t n = a.batch;
    const at::Tensor ints = new_tensor({3 * n + 2}, at::kInt, device);
    const at::Tensor cu = part_of(ints, 0, n + 1), lens = part_of(ints, n + 1, n);
    const at::Tensor placed = part_of(ints, 2 * n + 1, n), count = part_of(ints, 3 * n + 1, 1);
    a.slots = reinterpret_cast<long long*>(slots.data_ptr());
    a.cu_seqlens = static_cast<int*>(cu.data_ptr());
    a.seq_lens_out = static_cast<int*>(lens.data_ptr());
    a.free_count_out = static_cast<int*>(count.data_ptr());
    a.placed = static_cast<int*>(placed.data_ptr());
    void* stream = stream_of(device);
    if (without_gil([&] { return g.plan(&a, stream); }) != APEX_ATTN_OK) return nullptr;
    return wrapped({slots, cu, lens, count, placed});
  });
}

// (...): (seq_lens, free_count)
PyObject* release(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 6 || !g.release) return nullptr;
    apex_attn_kv_plan_args a{};
    int device = -1;
    if (!bookkeeping_args(a, o, false, device)) return nullptr;
    const at::Tensor both = new_tensor({(int64_t)a.batch + 1}, at::kInt, device);
    const at::Tensor lens = part_of(both, 0, a.batch), count = part_of(both, a.batch, 1);
    a.seq_lens_out = static_cast<int*>(lens.data_ptr());
    a.free_count_out = static_cast<int*>(count.data_ptr());
    void* stream = stream_of(device);
    if (without_gil([&] { return g.release(&a, stream); }) != APEX_ATTN_OK) return nullptr;
    return wrapped({lens, count});
  });
}

// (plan, release, append, workspace_bytes, attend): addresses of the C functions, 0 to unset
PyObject* init(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "init takes five addresses");
    return nullptr;
  }
  void* at[5];
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(o[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g.plan = reinterpret_cast<decltype(g.plan)>(at[0]);
  g.release = reinterpret_cast<decltype(g.release)>(at[1]);
  g.append = reinterpret_cast<decltype(g.append)>(at[2]);
  g.workspace_bytes = reinterpret_cast<decltype(g.workspace_bytes)>(at[3]);
  g.attend = reinterpret_cast<decltype(g.attend)>(at[4]);
  Py_RETURN_NONE;
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"init", fast(init), METH_FASTCALL, nullptr},
                         {"attend", fast(attend), METH_FASTCALL, nullptr},
                         {"append", fast(append), METH_FASTCALL, nullptr},
                         {"plan", fast(plan), METH_FASTCALL, nullptr},
                         {"release", fast(release), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#ifndef APEX_CALLS_KEY
#error "APEX_CALLS_KEY names the torch and Python versions that this is compiled against"
#endif

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", APEX_CALLS_KEY) < 0) Py_CLEAR(m);
  return m;
}
