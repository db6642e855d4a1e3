// The short way from Python to the calls that a decoder makes once per layer and
// token: kv8_append, attention_kv8 and sample.
//
// Through ctypes such a call spends 12 to 18 us on the host, more than its kernel runs
// in a small batch. Here the arguments are looked at in C++: a call whose every
// argument is as the entry point needs it, on the current device, is made at once
// (5 to 8 us). Anything else returns None, and ops.py goes its own way: it finds the same
// things wrong, says what, and raises; so messages and rules have one home.
//
// An extension module of the torch that it was compiled with (ops.py imports it if it
// is there); the entry points themselves come from libwbk.so by address.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "wbk.h"

namespace {

decltype(&wbk_kv8_append) g_append = nullptr;
decltype(&wbk_attention_kv8) g_attention = nullptr;
decltype(&wbk_attention_kv8_ws_bytes) g_ws_bytes = nullptr;
decltype(&wbk_sample) g_sample = nullptr;

// A tensor argument, or nullptr.
const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

int dtype16(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? WBK_DT_F16 : t.scalar_type() == at::kBFloat16 ? WBK_DT_BF16 : -1;
}

// A [B, H, S, D] view on CUDA device `index` with a contiguous last dimension; strides of its first three.
bool bhsd(const at::Tensor& t, int index, int64_t* strides) {
  if (!t.is_cuda() || t.get_device() != index || t.dim() != 4 || t.stride(3) != 1) return false;
  for (int i = 0; i < 3; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
  return true;
}

bool plain(const at::Tensor* t, int index, at::ScalarType type, int64_t numel) {
  return t != nullptr && t->is_cuda() && t->get_device() == index && t->scalar_type() == type && t->dim() == 1 &&
         t->size(0) == numel && t->is_contiguous();
}

int format(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "e4m3") == 0) return WBK_FMT_E4M3;
    if (PyUnicode_CompareWithASCIIString(o, "e5m2") == 0) return WBK_FMT_E5M2;
  }
  return -1;
}

struct Cache {
  const at::Tensor *k, *v, *ks, *vs, *table, *lens;
  int fmt;
  int64_t pages, heads, block, width, table_stride;
};

// k_cache, v_cache, k_scale, v_scale, block_table, seq_lens as args[0 .. 5].
bool cache_of(PyObject* const* args, PyObject* fmt, int index, int64_t batch, int64_t head_dim, Cache& c) {
  c.k = tensor(args[0]), c.v = tensor(args[1]), c.ks = tensor(args[2]), c.vs = tensor(args[3]);
  c.table = tensor(args[4]), c.lens = tensor(args[5]);
  c.fmt = format(fmt);
  if (c.fmt < 0 || c.k == nullptr || c.v == nullptr || c.ks == nullptr || c.vs == nullptr || c.table == nullptr) return false;
  const at::ScalarType f8 = c.fmt == WBK_FMT_E4M3 ? at::kFloat8_e4m3fn : at::kFloat8_e5m2;
  for (const at::Tensor* t : {c.k, c.v}) {
    const at::ScalarType type = t->scalar_type();
    if (!t->is_cuda() || t->get_device() != index || t->dim() != 4 || !t->is_contiguous() ||
        (type != f8 && type != at::kByte && type != at::kChar))
      return false;
  }
  if (c.k->sizes() != c.v->sizes() || c.k->size(3) != head_dim) return false;
  c.pages = c.k->size(0), c.heads = c.k->size(1), c.block = c.k->size(2);
  for (const at::Tensor* t : {c.ks, c.vs})
    if (!t->is_cuda() || t->get_device() != index || t->scalar_type() != at::kFloat || t->dim() != 2 ||
        t->size(0) != c.pages || t->size(1) != c.heads || !t->is_contiguous())
      return false;
  if (!c.table->is_cuda() || c.table->get_device() != index || c.table->scalar_type() != at::kInt || c.table->dim() != 2 ||
      c.table->size(0) != batch)
    return false;
  c.width = c.table->size(1);
  if (c.width > 1 && c.table->stride(1) != 1) return false;
  c.table_stride = batch > 1 ? c.table->stride(0) : c.width;
  return plain(c.lens, index, at::kInt, batch);
}

void* stream_of(int index) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index)).stream(); }

// bind(addresses of wbk_kv8_append, wbk_attention_kv8, wbk_attention_kv8_ws_bytes, wbk_sample)
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* at[4];
  if (n != 4) return PyErr_Format(PyExc_TypeError, "bind takes 4 addresses");
  for (int i = 0; i < 4; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "null address");
  }
  std::memcpy(&g_append, &at[0], sizeof(void*));
  std::memcpy(&g_attention, &at[1], sizeof(void*));
  std::memcpy(&g_ws_bytes, &at[2], sizeof(void*));
  std::memcpy(&g_sample, &at[3], sizeof(void*));
  Py_RETURN_NONE;
}

// kv8_append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, new_lens, fmt) -> status or None
PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const at::Tensor *k, *v;
  if (n != 10 || g_append == nullptr || (k = tensor(args[0])) == nullptr || (v = tensor(args[1])) == nullptr || !k->is_cuda()) Py_RETURN_NONE;
  const int index = c10::cuda::current_device(), dt = dtype16(*k);
  int64_t strides[6];
  Cache c;
  if (dt < 0 || v->scalar_type() != k->scalar_type() || !bhsd(*k, index, strides) || !bhsd(*v, index, strides + 3) ||
      k->sizes() != v->sizes() || !cache_of(args + 2, args[9], index, k->size(0), k->size(3), c) || c.heads != k->size(1))
    Py_RETURN_NONE;
  const at::Tensor* fresh = nullptr;
  if (args[8] != Py_None && !plain(fresh = tensor(args[8]), index, at::kInt, k->size(0))) Py_RETURN_NONE;
  return PyLong_FromLong(g_append(
      k->data_ptr(), v->data_ptr(), dt, k->size(0), k->size(1), k->size(2), k->size(3), strides, c.fmt, c.k->data_ptr(),
      c.v->data_ptr(), static_cast<float*>(c.ks->data_ptr()), static_cast<float*>(c.vs->data_ptr()), c.pages, c.block,
      static_cast<const int32_t*>(c.table->data_ptr()), c.width, c.table_stride,
      static_cast<const int32_t*>(c.lens->data_ptr()),
      fresh != nullptr ? static_cast<const int32_t*>(fresh->data_ptr()) : nullptr,
      static_cast<wbk_stream_t>(stream_of(index))));
}

// attention_kv8(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, q_lens, causal, scale, fmt, out, workspace,
// shared) -> output, status (an int) or None. shared: a list with each device's shared workspace, or None in its place.
PyObject* py_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const at::Tensor* q;
  if (n != 14 || g_attention == nullptr || (q = tensor(args[0])) == nullptr || !q->is_cuda()) Py_RETURN_NONE;
  const int index = c10::cuda::current_device(), dt = dtype16(*q);
  int64_t strides[6];
  Cache c;
  if (dt < 0 || !bhsd(*q, index, strides) || !cache_of(args + 1, args[10], index, q->size(0), q->size(3), c) || c.heads == 0 ||
      q->size(1) % c.heads != 0)
    Py_RETURN_NONE;
  const at::Tensor *q_lens = nullptr, *ws;
  if (args[7] != Py_None && !plain(q_lens = tensor(args[7]), index, at::kInt, q->size(0))) Py_RETURN_NONE;
  double scale;
  if (args[9] == Py_None) scale = c.k->size(3) == 64 ? 0.125 : 1.0 / std::sqrt(static_cast<double>(q->size(3)));
  else if (PyFloat_Check(args[9])) scale = PyFloat_AS_DOUBLE(args[9]);
  else Py_RETURN_NONE;
  PyObject* w = args[12];
  if (w == Py_None) {
    if (!PyList_Check(args[13]) || index >= PyList_GET_SIZE(args[13])) Py_RETURN_NONE;
    w = PyList_GET_ITEM(args[13], index);
  }
  if ((ws = tensor(w)) == nullptr || !ws->is_cuda() || ws->get_device() != index || !ws->is_contiguous()) Py_RETURN_NONE;
  const int64_t B = q->size(0), H = q->size(1), T = q->size(2), D = q->size(3);
  if (static_cast<int64_t>(ws->nbytes()) < g_ws_bytes(B, H, c.heads, T, D)) Py_RETURN_NONE;
  at::Tensor made;
  const at::Tensor* out;
  if (args[11] == Py_None) {
    made = at::empty(q->sizes(), q->options().requires_grad(false));
    out = &made;
    strides[3] = H * T * D, strides[4] = T * D, strides[5] = D;
  } else {
    out = tensor(args[11]);
    if (out == nullptr || out->scalar_type() != q->scalar_type() || !bhsd(*out, index, strides + 3) || out->sizes() != q->sizes())
      Py_RETURN_NONE;
  }
  const int causal = PyObject_IsTrue(args[8]);
  if (causal < 0) return nullptr;
  const int status = g_attention(
      q->data_ptr(), out->data_ptr(), dt, B, H, c.heads, T, D, strides, c.fmt, c.k->data_ptr(), c.v->data_ptr(),
      static_cast<const float*>(c.ks->data_ptr()), static_cast<const float*>(c.vs->data_ptr()), c.pages, c.block,
      static_cast<const int32_t*>(c.table->data_ptr()), c.width, c.table_stride,
      static_cast<const int32_t*>(c.lens->data_ptr()),
      q_lens != nullptr ? static_cast<const int32_t*>(q_lens->data_ptr()) : nullptr, causal, static_cast<float>(scale),
      ws->data_ptr(), static_cast<int64_t>(ws->nbytes()), static_cast<wbk_stream_t>(stream_of(index)));
  if (status != WBK_OK) return PyLong_FromLong(status);
  if (args[11] == Py_None) return THPVariable_Wrap(std::move(made));
  Py_INCREF(args[11]);
  return args[11];
}

// A setting of sample(): a number >= 0 or a device array. False: neither.
bool setting(PyObject* o, int index, at::ScalarType type, int64_t rows, double& all, const void*& row) {
  row = nullptr;
  all = 0.0;
  if (const at::Tensor* t = tensor(o)) {
    if (!plain(t, index, type, rows)) return false;
    row = t->data_ptr();
    return true;
  }
  if (PyFloat_Check(o)) all = PyFloat_AS_DOUBLE(o);
  else if (PyLong_Check(o)) {
    int overflow;
    const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (overflow != 0) return false;
    all = static_cast<double>(x);
  } else {
    return false;
  }
  return all >= 0.0 && all <= 2147483647.0;
}

// sample(logits, noise, temperature, top_k, top_p, min_p) -> (tokens, logprobs), status (an int) or None
PyObject* py_sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const at::Tensor *x, *e;
  if (n != 6 || g_sample == nullptr || (x = tensor(args[0])) == nullptr || (e = tensor(args[1])) == nullptr || !x->is_cuda()) Py_RETURN_NONE;
  const int index = c10::cuda::current_device();
  const at::ScalarType type = x->scalar_type();
  const int dt = type == at::kFloat ? WBK_DT_F32 : dtype16(*x);
  if (dt < 0 || !x->is_cuda() || x->get_device() != index || x->dim() != 2 || !e->is_cuda() || e->get_device() != index ||
      e->scalar_type() != at::kFloat || e->sizes() != x->sizes())
    Py_RETURN_NONE;
  const int64_t rows = x->size(0), vocab = x->size(1);
  if (rows == 0 || vocab < 2 || x->stride(1) != 1 || e->stride(1) != 1) Py_RETURN_NONE;
  double t_all, k_all, p_all, m_all;
  const void *t_row, *k_row, *p_row, *m_row;
  if (!setting(args[2], index, at::kFloat, rows, t_all, t_row) || !setting(args[3], index, at::kInt, rows, k_all, k_row) ||
      !setting(args[4], index, at::kFloat, rows, p_all, p_row) || !setting(args[5], index, at::kFloat, rows, m_all, m_row) ||
      k_all != static_cast<double>(static_cast<int>(k_all)))
    Py_RETURN_NONE;
  at::Tensor tokens = at::empty({rows}, x->options().dtype(at::kLong).requires_grad(false));
  at::Tensor logprobs = at::empty({rows}, x->options().dtype(at::kFloat).requires_grad(false));
  const int status = g_sample(
      x->data_ptr(), dt, rows, vocab, rows > 1 ? x->stride(0) : vocab, static_cast<const float*>(e->data_ptr()),
      rows > 1 ? e->stride(0) : vocab, static_cast<const float*>(t_row), static_cast<const int32_t*>(k_row),
      static_cast<const float*>(p_row), static_cast<const float*>(m_row), static_cast<float>(t_all), static_cast<int>(k_all),
      static_cast<float>(p_all), static_cast<float>(m_all), static_cast<int64_t*>(tokens.data_ptr()),
      static_cast<float*>(logprobs.data_ptr()), static_cast<wbk_stream_t>(stream_of(index)));
  if (status != WBK_OK) return PyLong_FromLong(status);
  PyObject* pair = PyTuple_New(2);
  if (pair == nullptr) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(logprobs)));
  return pair;
}

// No C++ exception (an allocation that fails, a CUDA error) leaves through the C interface.
template <PyObject* (*kFn)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return kFn(self, args, n);
  } catch (const c10::OutOfMemoryError&) {
    Py_RETURN_NONE;  // the other way meets it too, and raises torch's own exception
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyCFunction fast(PyObject* (*fn)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn));
}

PyMethodDef g_methods[] = {
    {"bind", fast(guarded<py_bind>), METH_FASTCALL, "Addresses of the entry points."},
    {"kv8_append", fast(guarded<py_append>), METH_FASTCALL, "Status, or None: not a call for the short way."},
    {"attention_kv8", fast(guarded<py_attention>), METH_FASTCALL, "Output, status, or None: not a call for the short way."},
    {"sample", fast(guarded<py_sample>), METH_FASTCALL, "(tokens, logprobs), status, or None: not a call for the short way."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_wbk_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__wbk_calls(void) {
  PyObject* m = PyModule_Create(&g_module);
  // the interpreter and the torch whose internals this was compiled against: the loader uses it with no other
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", WBK_CALLS_FOR) != 0) Py_CLEAR(m);
  return m;
}
