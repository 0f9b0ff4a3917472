// CPython binding of the hk_* entry points that a decode step calls over and over.
//
// A launch costs the host about 2 us; through ctypes the same call cost 10-15 us more (one c_void_p object per tensor, the
// argtypes conversion of 20-30 arguments, a torch Stream object per call), which made every decode call host-bound
// (the KDA layer of one token: 17.2 us per call around a 5.4 us kernel; with this binding 5.5 us).  Here a call is one
// METH_FASTCALL function: tensors are unwrapped to their addresses and the numbers converted straight into the C call.
//
// Conversion rules, by the C type of the parameter:
//   pointer        tensor (or another object with data_ptr()) -> its address, None -> NULL; a tensor that has no address
//                  (sparse, wrapped by a transform) raises the RuntimeError of Tensor.data_ptr()
//   void* stream   (last parameter of a launcher) None -> torch's current stream, torch Stream -> its handle
//   int            int / bool; a tensor gives the dtype tag HK_F16 / HK_BF16 / HK_F32
//   int64_t        int; a [rows][512] tensor gives its row count, 0 if it is not laid out that way
//   size_t         int; a tensor gives its element count (byte workspaces), None gives 0
//   float          number
// The functions return what the C function returns (launchers: the hk_status).  The addresses come from the library that
// the Python layer loaded (bind), so that both sides drive the same build.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/Exception.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/helios_b200.h"

namespace {

bool bad_arg(const char* what) {
  PyErr_SetString(PyExc_TypeError, what);
  return false;
}

bool number(PyObject* o, long long& v) {
  v = PyLong_AsLongLong(o);
  return !(v == -1 && PyErr_Occurred());
}

template <class T>
bool convert(PyObject* o, T& v) {
  if constexpr (std::is_pointer_v<T>) {
    if (o == Py_None) {
      v = nullptr;
      return true;
    }
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      // what the call writes is asked for as such: a lazily cloned tensor gets memory of its own first
      if constexpr (std::is_const_v<std::remove_pointer_t<T>>) v = reinterpret_cast<T>(t.const_data_ptr());
      else v = reinterpret_cast<T>(t.mutable_data_ptr());
      return true;
    }
    PyObject* a = PyObject_CallMethod(o, "data_ptr", nullptr);
    if (!a) return false;
    v = reinterpret_cast<T>(PyLong_AsVoidPtr(a));
    Py_DECREF(a);
    return !PyErr_Occurred();
  } else if constexpr (std::is_floating_point_v<T>) {
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) return false;
    v = static_cast<T>(d);
    return true;
  } else {
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      if constexpr (std::is_same_v<T, int>) {
        switch (t.scalar_type()) {
          case at::kHalf: v = HK_F16; return true;
          case at::kBFloat16: v = HK_BF16; return true;
          case at::kFloat: v = HK_F32; return true;
          default: return bad_arg("tensor dtype: float16, bfloat16 or float32");
        }
      } else if constexpr (std::is_same_v<T, size_t>) {
        v = static_cast<T>(t.numel());
      } else {
        v = t.dim() >= 1 && t.numel() % 512 == 0 ? static_cast<T>(t.numel() / 512) : 0;
      }
      return true;
    }
    if constexpr (std::is_same_v<T, size_t>) {
      if (o == Py_None) {
        v = 0;
        return true;
      }
    }
    long long n;
    if (!number(o, n)) return false;
    if constexpr (std::is_same_v<T, int>) {
      if (n < INT32_MIN || n > INT32_MAX) return bad_arg("integer argument out of range");
    }
    v = static_cast<T>(n);
    return true;
  }
}

bool convert_stream(PyObject* o, void*& v) {
  if (o == Py_None) {
    try {
      v = c10::cuda::getCurrentCUDAStream().stream();
    } catch (const std::exception&) {
      PyErr_SetString(PyExc_RuntimeError, "helios_glm53flash_b200 needs a CUDA device (sm_100a); there is no CPU path");
      return false;
    }
    return true;
  }
  PyObject* h = PyObject_GetAttrString(o, "cuda_stream");
  if (!h) return false;
  v = PyLong_AsVoidPtr(h);
  Py_DECREF(h);
  return !PyErr_Occurred();
}

template <bool STREAM, size_t I, size_t N, class T>
bool convert_at(PyObject* o, T& v) {
  if constexpr (STREAM && I + 1 == N) return convert_stream(o, v);
  else return convert(o, v);
}

template <bool STREAM, class R, class... A, size_t... I>
PyObject* call(R (*fn)(A...), PyObject* const* args, std::index_sequence<I...>) {
  std::tuple<std::remove_const_t<A>...> v;
  try {
    if (!(convert_at<STREAM, I, sizeof...(A)>(args[I], std::get<I>(v)) && ...)) return nullptr;
  } catch (const c10::Error& e) {          // a tensor without an address: sparse, wrapped by vmap, ...
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  R r;
  if constexpr (STREAM) {
    Py_BEGIN_ALLOW_THREADS;      // a launch may wait for room in the stream's queue
    r = fn(std::get<I>(v)...);
    Py_END_ALLOW_THREADS;
  } else {
    r = fn(std::get<I>(v)...);
  }
  if constexpr (std::is_same_v<R, size_t>) return PyLong_FromSize_t(r);
  else return PyLong_FromLong(r);
}

template <class F>
struct Entry;
template <class R, class... A>
struct Entry<R (*)(A...)> {
  template <bool STREAM>
  static PyObject* run(R (*fn)(A...), const char* name, PyObject* const* args, Py_ssize_t n) {
    if (!fn) {
      PyErr_SetString(PyExc_RuntimeError, "the binding is not bound to the library");
      return nullptr;
    }
    if (n != (Py_ssize_t)sizeof...(A))
      return PyErr_Format(PyExc_TypeError, "%s takes %d arguments, %d given", name, (int)sizeof...(A), (int)n);
    return call<STREAM>(fn, args, std::index_sequence_for<A...>{});
  }
};

// every entry point: X(name, ends in a stream)
#define HK_ENTRIES(X)                                                                                                       \
  X(hk_conv1d_update, true) X(hk_kda_recurrent, true) X(hk_kda_decode_step, true) X(hk_kda_decode_layer, true)               \
  X(hk_kda_dispatch_is_chunked, false) X(hk_kda_chunked_workspace_bytes, false) X(hk_kda_chunked_prefill, true)              \
  X(hk_kda_chunked_prefill_gated, true) X(hk_kda_transpose_cast, true) X(hk_kda_gate, true) X(hk_kda_prepare, true)          \
  X(hk_kda_cast_conv, true) X(hk_gated_rms_norm, true) X(hk_kpool_write, true) X(hk_indexer_score, true)                     \
  X(hk_indexer_score_legacy, true) X(hk_dsa_topk, true) X(hk_dsa_topk_expand, true) X(hk_indexer_select, true)               \
  X(hk_pool_expand, true) X(hk_mla_partial_bytes, false) X(hk_mla_auto_splits, false) X(hk_mla_sparse, true)                 \
  X(hk_mla_sparse_static, true) X(hk_mla_dense, true) X(hk_mla_dense_partial, true) X(hk_mla_dense_partial_ws, true)         \
  X(hk_lse_combine, true) X(hk_q_latent, true) X(hk_o_absorb, true) X(hk_wuv_transpose, true) X(hk_o_absorb_t, true)         \
  X(hk_q_latent_beside, true) X(hk_o_absorb_beside, true) X(hk_kda_decode_layer_beside, true)                                \
  X(hk_mla_cache_append, true) X(hk_layernorm_f16, true) X(hk_mla_decode_prologue, true) X(hk_mla_window, true)              \
  X(hk_mla8_append, true) X(hk_mla8_read, true) X(hk_mla8_dense, true) X(hk_mla8_sparse, true)                                \
  X(hk_mla8_dense_workspace_bytes, false) X(hk_mla8_sparse_workspace_bytes, false)                                        \
  X(hk_mla_window_keys, false) X(hk_mla_window_workspace_bytes, false)

#define X(name, stream)                                                                      \
  decltype(&::name) p_##name = nullptr;                                                      \
  PyObject* py_##name(PyObject*, PyObject* const* args, Py_ssize_t n) {                      \
    return Entry<decltype(&::name)>::run<stream>(p_##name, #name, args, n);                  \
  }
HK_ENTRIES(X)
#undef X

// bind(dict name -> address)
PyObject* py_bind(PyObject*, PyObject* d) {
  if (!PyDict_Check(d)) {
    bad_arg("bind: a dict of addresses");
    return nullptr;
  }
#define X(name, stream)                                                                       \
  {                                                                                           \
    PyObject* a = PyDict_GetItemString(d, #name);                                             \
    if (!a) return PyErr_Format(PyExc_KeyError, "%s", #name);                                 \
    void* p = PyLong_AsVoidPtr(a);                                                            \
    if (PyErr_Occurred()) return nullptr;                                                     \
    p_##name = reinterpret_cast<decltype(p_##name)>(p);                                       \
  }
  HK_ENTRIES(X)
#undef X
  Py_RETURN_NONE;
}

// the current device, asked for once a call; -1: there is none
int device_now() {
  static const int devices = c10::cuda::device_count();
  return devices > 0 ? c10::cuda::current_device() : -1;
}
// an address of the host, or of another GPU than the one that the call runs on, would be a fault there
bool elsewhere(const at::Tensor& t, int device) { return device >= 0 && (!t.is_cuda() || t.device().index() != device); }

// None, or contiguous, of the type (h: float16, f: float32, i: int32, l: int64) and of as many elements as the call reads or writes, or more
bool check_tensor(PyObject* o, char type, const char* name, long long least, int device) {
  if (o == Py_None) return true;
  const auto want = type == 'h' ? at::kHalf : type == 'f' ? at::kFloat : type == 'i' ? at::kInt : at::kLong;
  if (THPVariable_Check(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() == want && t.is_contiguous() && t.numel() >= least && !elsewhere(t, device)) return true;
  }
  PyErr_Format(PyExc_ValueError, "%s: a contiguous tensor of %s on the current CUDA device, of %lld elements or more", name,
               type == 'h' ? "float16" : type == 'f' ? "float32" : type == 'i' ? "int32" : "int64", least);
  return false;
}
// (types, names, tensor, elements, tensor, elements, ...)
bool check_tensors(PyObject* const* args, Py_ssize_t n, int device) {
  Py_ssize_t len = 0;
  const char* types = n >= 2 && PyUnicode_Check(args[0]) ? PyUnicode_AsUTF8AndSize(args[0], &len) : nullptr;
  if (!types || !PyTuple_Check(args[1]) || PyTuple_GET_SIZE(args[1]) != len || n != 2 + 2 * len) return bad_arg("types, names, then a tensor and a size each");
  for (Py_ssize_t k = 0; k < len; k++) {
    long long least;
    const char* name = PyUnicode_AsUTF8(PyTuple_GET_ITEM(args[1], k));
    if (!name || !number(args[3 + 2 * k], least) || !check_tensor(args[2 + 2 * k], types[k], name, least, device)) return false;
  }
  return true;
}
PyObject* py_tensors(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (!check_tensors(args, n, device_now())) return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

// The arguments that an 8-bit latent cache's tensors (ckv8, scales, block_table or None) stand for.  What the library cannot see from addresses is
// checked here.
struct Cache8 {
  int dtype;
  long long n_blocks, block, stride = 0, seqs = 1;
};
bool cache8_of(PyObject* const* args, int device, Cache8& v) {
  auto refuse = [](const char* what) {
    PyErr_SetString(PyExc_ValueError, what);
    return false;
  };
  if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]) || !(args[2] == Py_None || THPVariable_Check(args[2]))) return bad_arg("cache8: the cache's tensors");
  const at::Tensor &c = THPVariable_Unpack(args[0]), &s = THPVariable_Unpack(args[1]);
  const bool i8 = c.scalar_type() == at::kChar;
  if ((!i8 && c.scalar_type() != at::kFloat8_e4m3fn) || c.dim() != 3 || c.size(2) != 512 || !c.is_contiguous())
    return refuse("ckv8: a contiguous [n_blocks, block, 512] tensor of int8 or float8_e4m3fn");
  if (c.size(1) > INT32_MAX) return refuse("ckv8: blocks of at most 128 tokens");
  if (s.scalar_type() != at::kFloat || s.numel() != c.size(0) || !s.is_contiguous()) return refuse("scales: a contiguous float32 tensor, one a block");
  if (elsewhere(c, device) || elsewhere(s, device) || (args[2] != Py_None && elsewhere(THPVariable_Unpack(args[2]), device)))
    return refuse("the 8-bit cache's tensors: on the current CUDA device");
  v.dtype = i8 ? HK_I8 : HK_E4M3;
  v.n_blocks = c.size(0);
  v.block = c.size(1);
  if (args[2] != Py_None) {
    const at::Tensor& t = THPVariable_Unpack(args[2]);
    if (t.scalar_type() != at::kInt || t.dim() < 1 || t.dim() > 2 || !t.is_contiguous() || t.numel() == 0)
      return refuse("block_table: a contiguous [n_seqs, blocks of a sequence] tensor of int32");
    v.stride = t.size(-1);
    v.seqs = t.numel() / v.stride;
    if (v.stride > INT32_MAX || v.seqs > INT32_MAX) return refuse("block_table: at most 2^31 - 1 sequences and blocks of one");
  }
  return true;
}

// cache8(ckv8, scales, block_table or None[, what check_tensors takes]) -> (dtype tag, n_blocks, block, table stride, n_seqs)
PyObject* py_cache8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n < 3) {
    bad_arg("cache8: the cache's tensors");
    return nullptr;
  }
  try {
    const int device = device_now();
    Cache8 v;
    if (!cache8_of(args, device, v) || (n > 3 && !check_tensors(args + 3, n - 3, device))) return nullptr;
    return Py_BuildValue("(iLLLL)", v.dtype, v.n_blocks, v.block, v.stride, v.seqs);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// append8(ckv8, scales, block_table, kv_pre, ln_w, pos, n, eps, n_seqs, seq_start, ckv_new, stream): the checks and hk_mla8_append in one call (a
// launch of a few rows takes less time than the host: 3.5 us a call as two, 2.9 as one, 2.75 in a graph)
PyObject* py_append8(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  if (n_args != 12 || !p_hk_mla8_append) {
    bad_arg("append8: 12 arguments, of a bound binding");
    return nullptr;
  }
  PyObject *kv_pre = args[3], *ln_w = args[4], *pos = args[5], *seq_start = args[9], *ckv_new = args[10];
  try {
    const int device = device_now();
    Cache8 c;
    int n, seqs;
    float eps;
    void* stream;
    const float* x;
    const void* w;
    void *ckv8, *new_rows;
    float* scales;
    const int *table, *starts, *at;
    if (!convert(args[6], n) || !convert(args[7], eps) || !convert(args[8], seqs) || !cache8_of(args, device, c) ||
        !check_tensor(kv_pre, 'f', "kv_pre", n * 512LL, device) || !check_tensor(ln_w, 'h', "ln_w", 512, device) ||
        !check_tensor(pos, 'i', "pos", seqs, device) || !check_tensor(seq_start, 'i', "seq_start", seqs + 1LL, device) ||
        !check_tensor(ckv_new, 'h', "ckv_new", n * 512LL, device))
      return nullptr;
    if (seqs > c.seqs) {
      PyErr_SetString(PyExc_ValueError, "block_table: fewer sequences than n_seqs");
      return nullptr;
    }
    if (!convert(kv_pre, x) || !convert(ln_w, w) || !convert(args[0], ckv8) || !convert(args[1], scales) || !convert(args[2], table) ||
        !convert(seq_start, starts) || !convert(pos, at) || !convert(ckv_new, new_rows) || !convert_stream(args[11], stream))
      return nullptr;
    int status;
    Py_BEGIN_ALLOW_THREADS;      // as in call
    status = p_hk_mla8_append(x, w, ckv8, scales, c.dtype, c.n_blocks, (int)c.block, table, (int)c.stride, seqs, starts, at, n, eps, new_rows, stream);
    Py_END_ALLOW_THREADS;
    return PyLong_FromLong(status);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// scratch(nbytes, tensor) -> a byte tensor of torch's allocator on the tensor's device (torch.empty from Python costs twice the time)
PyObject* py_scratch(PyObject*, PyObject* const* args, Py_ssize_t n) {
  long long bytes;
  if (n != 2 || !THPVariable_Check(args[1])) {
    bad_arg("scratch: a size and a tensor");
    return nullptr;
  }
  if (!number(args[0], bytes)) return nullptr;
  try {
    return THPVariable_Wrap(at::empty({bytes < 256 ? 256 : bytes}, THPVariable_Unpack(args[1]).options().dtype(at::kByte).requires_grad(false)));
  } catch (const std::exception& e) {          // out of memory among them
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define X(name, stream) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr},
PyMethodDef methods[] = {HK_ENTRIES(X){"cache8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_cache8)), METH_FASTCALL, nullptr},
                         {"append8", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_append8)), METH_FASTCALL, nullptr},
                         {"tensors", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_tensors)), METH_FASTCALL, nullptr},
                         {"scratch", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_scratch)), METH_FASTCALL, nullptr},
                         {"bind", py_bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
#undef X

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "native call path of the hk_* entry points", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module); }
