// Python calls of the cache, attention and norm entry points, as a CPython module.
//
// A decode step makes these calls for every layer, and their kernels take a few microseconds: reading
// a tensor's sizes and strides, allocating outputs and filling a struct of 30 fields from Python takes
// longer than that. Each function here does the same for arguments in the usual form and launches on
// the current stream. For any others it returns None, and the caller takes the way through the builders
// of ops.py, which knows every form and says what is wrong. A status other than 0 is returned as an int.
//
// (Host time of a call in us, here against through the builders: norm with a residual to e4m3, 5.7 against
// 13.5; attention with log-sum-exps 5.4 against 13.0; append of slices 6.5 against 12.5; gather 5.2 against
// 11.3. The launch itself takes 2.7.)

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/sonic_b200.h"

namespace {

// entry points of the library that Python loaded
decltype(&sonic_residual_norm) residual_norm_entry;
decltype(&sonic_cache_append) cache_append_entry;
decltype(&sonic_cache_gather) cache_gather_entry;
decltype(&sonic_paged_attention) paged_attention_entry;

struct Absent {};  // an argument in another form than the usual one

// the address that a ctypes struct or a device buffer has, from an int
template <typename T>
T* address(PyObject* o) {
  T* p = static_cast<T*>(PyLong_AsVoidPtr(o));
  if (!p && PyErr_Occurred()) throw python_error();
  return p;
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Absent();
  }
  return v;
}

const at::Tensor& tensor(PyObject* o, const at::Device& device) {
  if (!THPVariable_Check(o)) throw Absent();
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided || t.device() != device) throw Absent();
  return t;
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return SONIC_DTYPE_BF16;
    case at::kHalf: return SONIC_DTYPE_F16;
    case at::kFloat: return SONIC_DTYPE_F32;
    case at::kFloat8_e4m3fn: return SONIC_DTYPE_E4M3;
    default: throw Absent();
  }
}

// the device of index `o`, where it is the current one
at::Device current(PyObject* o) {
  const int64_t index = integer(o);
  if (index != c10::cuda::current_device()) throw Absent();
  return at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(index));
}
void* stream_of(const at::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(device));
}

// [tokens, heads, head_dim] with a unit inner stride: returns the tokens
int64_t token_rows(const at::Tensor& t, int64_t heads, int64_t dim, int64_t& token_stride, int64_t& head_stride) {
  if (t.dim() != 3 || t.size(1) != heads || t.size(2) != dim || t.stride(2) != 1 || t.size(0) > INT32_MAX) throw Absent();
  token_stride = t.stride(0), head_stride = t.stride(1);
  return t.size(0);
}

const int32_t* index_vector(PyObject* o, int64_t size, const at::Device& device) {
  const at::Tensor& t = tensor(o, device);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != size || (size > 1 && t.stride(0) != 1)) throw Absent();
  return static_cast<const int32_t*>(t.data_ptr());
}

// page table, and where they are not null lengths and cu_seqlens (which may be None)
int64_t sequences(SonicSequences& s, int64_t tokens, PyObject* table_object, PyObject* lengths, PyObject* cu, const at::Device& device) {
  const at::Tensor& table = tensor(table_object, device);
  if (table.scalar_type() != at::kInt || table.dim() != 2 || (table.stride(1) != 1 && table.size(1) > 1) ||
      table.size(0) >= INT32_MAX || table.size(1) > INT32_MAX)
    throw Absent();
  const int64_t requests = table.size(0);
  s.requests = static_cast<int32_t>(requests);
  s.tokens = static_cast<int32_t>(tokens);
  s.page_table = static_cast<const int32_t*>(table.data_ptr());
  s.table_stride = table.stride(0);
  s.table_width = static_cast<int32_t>(table.size(1));
  s.lengths = s.cu_seqlens = nullptr;
  if (lengths) {
    s.lengths = index_vector(lengths, requests, device);
    if (cu != Py_None)
      s.cu_seqlens = index_vector(cu, requests + 1, device);
    else if (requests == 0 || tokens % requests)
      throw Absent();
  }
  return requests;
}

void activations(at::ScalarType t) {
  if (t != at::kBFloat16 && t != at::kHalf) throw Absent();
}

// norm(template, x, weight, residual or None) -> (out, scales or None, residual_out or None)
PyObject* norm(PyObject* const* v) {
  SonicResidualNormArgs a = *address<const SonicResidualNormArgs>(v[0]);
  if (!THPVariable_Check(v[2])) throw Absent();
  const at::Tensor& weight = THPVariable_Unpack(v[2]);
  const at::Device device = weight.device();
  if (!device.is_cuda() || device.index() != c10::cuda::current_device()) throw Absent();
  const at::ScalarType type = weight.scalar_type();
  const int64_t hidden = a.hidden;
  const auto rows_of = [&](PyObject* o, int64_t& stride) -> const at::Tensor& {
    const at::Tensor& t = tensor(o, device);
    if (t.dim() != 2 || t.size(1) != hidden || t.scalar_type() != type || (t.stride(1) != 1 && hidden > 1)) throw Absent();
    stride = t.stride(0);
    return t;
  };
  const at::Tensor& x = rows_of(v[1], a.x_stride);
  const int64_t rows = x.size(0);
  if (rows > INT32_MAX || weight.dim() != 1 || weight.size(0) != hidden || dtype_code(type) != a.dtype) throw Absent();
  a.rows = static_cast<int32_t>(rows);
  a.x = x.data_ptr();
  a.weight = weight.data_ptr();
  at::Tensor residual_out, scales;
  if (v[3] != Py_None) {
    const at::Tensor& residual = rows_of(v[3], a.residual_stride);
    if (residual.size(0) != rows) throw Absent();
    a.residual = residual.data_ptr();
    residual_out = empty({rows, hidden}, type, device);
    a.residual_out = residual_out.data_ptr();
    a.residual_out_stride = hidden;
  }
  const bool q8 = a.out_dtype == SONIC_DTYPE_E4M3;
  const at::Tensor out = empty({rows, hidden}, q8 ? at::kFloat8_e4m3fn : type, device);
  a.out = out.data_ptr();
  a.out_stride = hidden;
  if (q8) {
    scales = empty({rows, a.group ? (hidden + a.group - 1) / a.group : 1}, at::kFloat, device);
    a.scales = static_cast<float*>(scales.data_ptr());
  }
  if (const sonic_status status = residual_norm_entry(&a, stream_of(device))) return PyLong_FromLong(status);
  const auto wrap = [](const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); };
  PyObject* const items[3] = {wrap(out), wrap(scales), wrap(residual_out)};
  PyObject* const tuple = items[0] && items[1] && items[2] ? PyTuple_Pack(3, items[0], items[1], items[2]) : nullptr;
  for (PyObject* item : items) Py_XDECREF(item);
  return tuple;
}

// append(cache, device, flags, error, keys, values, page_table, lengths, cu_seqlens or None) -> status
PyObject* append(PyObject* const* v) {
  SonicCacheAppendArgs a = {};
  a.cache = *address<const SonicPagedCache>(v[0]);
  const at::Device device = current(v[1]);
  a.flags = static_cast<uint32_t>(integer(v[2]));
  a.error = address<uint32_t>(v[3]);
  const at::Tensor &keys = tensor(v[4], device), &values = tensor(v[5], device);
  activations(keys.scalar_type());
  if (values.scalar_type() != keys.scalar_type()) throw Absent();
  const int64_t tokens = token_rows(keys, a.cache.kv_heads, a.cache.head_dim, a.key_token_stride, a.key_head_stride);
  if (token_rows(values, a.cache.kv_heads, a.cache.head_dim, a.value_token_stride, a.value_head_stride) != tokens) throw Absent();
  sequences(a.sequences, tokens, v[6], v[7], v[8], device);
  a.dtype = dtype_code(keys.scalar_type());
  a.keys = keys.data_ptr();
  a.values = values.data_ptr();
  return PyLong_FromLong(cache_append_entry(&a, stream_of(device)));
}

// gather(cache, device, flags, error, page_table, starts, total, fp16) -> (keys, values)
PyObject* gather(PyObject* const* v) {
  SonicCacheGatherArgs a = {};
  a.cache = *address<const SonicPagedCache>(v[0]);
  const at::Device device = current(v[1]);
  a.flags = static_cast<uint32_t>(integer(v[2]));
  a.error = address<uint32_t>(v[3]);
  const int64_t total = integer(v[6]);
  if (total < 0 || total > INT32_MAX) throw Absent();
  const int64_t requests = sequences(a.sequences, total, v[4], nullptr, nullptr, device);
  a.starts = index_vector(v[5], requests + 1, device);
  const at::ScalarType type = v[7] == Py_True ? at::kHalf : at::kBFloat16;
  const at::Tensor keys = empty({total, a.cache.kv_heads, a.cache.head_dim}, type, device);
  const at::Tensor values = empty({total, a.cache.kv_heads, a.cache.head_dim}, type, device);
  a.dtype = dtype_code(type);
  a.keys = keys.data_ptr();
  a.values = values.data_ptr();
  if (const sonic_status status = cache_gather_entry(&a, stream_of(device))) return PyLong_FromLong(status);
  PyObject *const x = THPVariable_Wrap(keys), *const y = THPVariable_Wrap(values);
  PyObject* const tuple = x && y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x), Py_XDECREF(y);
  return tuple;
}

// attention(template, cache, device, workspace, bytes, queries, page_table, lengths, cu_seqlens or None,
// max_tokens, window or None, scale or None, logsumexp) -> out, or (out, lse)
PyObject* attention(PyObject* const* v) {
  SonicPagedAttentionArgs a = *address<const SonicPagedAttentionArgs>(v[0]);
  a.cache = *address<const SonicPagedCache>(v[1]);
  const at::Device device = current(v[2]);
  a.workspace = address<void>(v[3]);
  a.workspace_bytes = static_cast<size_t>(integer(v[4]));
  const at::Tensor& queries = tensor(v[5], device);
  activations(queries.scalar_type());
  const int64_t heads = a.q_heads, dim = a.cache.head_dim;
  const int64_t tokens = token_rows(queries, heads, dim, a.q_token_stride, a.q_head_stride);
  sequences(a.sequences, tokens, v[6], v[7], v[8], device);
  a.max_tokens = v[8] == Py_None ? 0 : static_cast<int32_t>(integer(v[9]));
  a.window = 0;
  if (v[10] != Py_None) {
    const int64_t window = integer(v[10]);
    if (window < 1 || window > INT32_MAX) throw Absent();
    a.window = static_cast<int32_t>(window);
  }
  if (v[11] != Py_None) {
    if (!PyFloat_Check(v[11])) throw Absent();
    a.scale = static_cast<float>(PyFloat_AS_DOUBLE(v[11]));
  }
  const bool logsumexp = v[12] == Py_True;
  if (!logsumexp && v[12] != Py_False) throw Absent();
  const at::Tensor out = empty({tokens, heads, dim}, queries.scalar_type(), device);
  at::Tensor lse;
  if (logsumexp) {
    lse = empty({tokens, heads}, at::kFloat, device);
    a.lse = static_cast<float*>(lse.data_ptr());
  }
  a.dtype = dtype_code(queries.scalar_type());
  a.queries = queries.data_ptr();
  a.out = out.data_ptr();
  a.out_token_stride = heads * dim;
  a.out_head_stride = dim;
  if (const sonic_status status = paged_attention_entry(&a, stream_of(device))) return PyLong_FromLong(status);
  PyObject* const x = THPVariable_Wrap(out);
  if (!logsumexp || !x) return x;
  PyObject* const y = THPVariable_Wrap(lse);
  PyObject* const tuple = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x), Py_XDECREF(y);
  return tuple;
}

template <PyObject* (*function)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, count);
    return nullptr;
  }
  if (!residual_norm_entry) {
    PyErr_SetString(PyExc_RuntimeError, "bind() comes first");
    return nullptr;
  }
  try {
    return function(args);
  } catch (const Absent&) {
    Py_RETURN_NONE;
  }
  END_HANDLE_TH_ERRORS
}

// bind(residual_norm, cache_append, cache_gather, paged_attention): the entry points' addresses
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 4) {
    PyErr_Format(PyExc_TypeError, "expected 4 arguments, got %zd", count);
    return nullptr;
  }
  void* at[4];
  for (int i = 0; i < 4; ++i) at[i] = address<void>(args[i]);
  residual_norm_entry = reinterpret_cast<decltype(residual_norm_entry)>(at[0]);
  cache_append_entry = reinterpret_cast<decltype(cache_append_entry)>(at[1]);
  cache_gather_entry = reinterpret_cast<decltype(cache_gather_entry)>(at[2]);
  paged_attention_entry = reinterpret_cast<decltype(paged_attention_entry)>(at[3]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"bind", fast(bind), METH_FASTCALL, nullptr},
    {"norm", fast(entry<norm, 4>), METH_FASTCALL, nullptr},
    {"append", fast(entry<append, 9>), METH_FASTCALL, nullptr},
    {"gather", fast(entry<gather, 8>), METH_FASTCALL, nullptr},
    {"attention", fast(entry<attention, 13>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "sonic_b200_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_sonic_b200_calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddIntConstant(m, "abi_version", SONIC_B200_ABI_VERSION)) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
