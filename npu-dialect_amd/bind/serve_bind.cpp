// serve_bind.cpp -- the serving entry points for Python: torch tensors to
// npu_memref descriptors in C++.
//
// A serving step calls these entry points once per layer and token with nine to
// eleven tensors each, and a small batch's kernels run for 3 to 5 us: packing the
// descriptors in Python took 12 us of a call, here they take less than one.
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/npu_amd.h"

namespace {

// The code of a type that an older torch does not name, by what this one calls it; -1: none.
int32_t newer_dtype(at::ScalarType type) {
  const char *name = c10::toString(type);
  if (!std::strcmp(name, "Float8_e4m3fn")) return NPU_E4M3;
  if (!std::strcmp(name, "Float8_e8m0fnu") || !std::strcmp(name, "Float4_e2m1fn_x2")) return NPU_U8;
  return -1;
}

// Descriptor of a tensor on the GPU (None: an operand that is not present, where
// that is allowed).  False with a Python error set.
bool describe(PyObject *o, const char *name, bool optional, npu_memref *m) {
  std::memset(m, 0, sizeof *m);
  if (o == Py_None && optional) {
    m->rank = 1;
    return true;
  }
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: expected a tensor, got %s", name, Py_TYPE(o)->tp_name);
    return false;
  }
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.is_cuda()) {  // a host pointer would fault in the kernel
    PyErr_Format(PyExc_ValueError, "%s: expected a tensor on the GPU, got one on %s", name, t.device().str().c_str());
    return false;
  }
  switch (t.scalar_type()) {
    case at::kFloat: m->dtype = NPU_F32; break;
    case at::kBFloat16: m->dtype = NPU_BF16; break;
    case at::kChar: m->dtype = NPU_I8; break;
    case at::kInt: m->dtype = NPU_I32; break;
    case at::kByte: m->dtype = NPU_U8; break;
    default:
      m->dtype = newer_dtype(t.scalar_type());
      if (m->dtype >= 0) break;
      PyErr_Format(PyExc_TypeError, "%s: unsupported tensor dtype %s", name, c10::toString(t.scalar_type()));
      return false;
  }
  if (t.dim() > NPU_MAX_RANK) {
    PyErr_Format(PyExc_ValueError, "%s: npu_memref holds at most rank %d", name, NPU_MAX_RANK);
    return false;
  }
  m->rank = (int32_t)t.dim();
  // (an empty tensor has no address, and none would mean an operand that is not present: the
  // entry point refuses its size)
  m->allocated = m->aligned = t.numel() > 0 ? t.data_ptr() : m;
  for (int d = 0; d < m->rank; ++d) {
    m->sizes[d] = t.size(d);
    m->strides[d] = t.stride(d);
  }
  return true;
}

struct Operand {
  const char *name;
  bool optional;
};
// The tensors' one device has to be the current one, which the kernels run on: another's memory
// may not be theirs to reach.  (ops[0] is never optional.)
template <int N>
bool on_current_device(PyObject *const *args, const Operand (&ops)[N]) {
  if (!THPVariable_Check(args[0]) || !THPVariable_Unpack(args[0]).is_cuda()) return true;  // describe() says so
  const c10::Device first = THPVariable_Unpack(args[0]).device();
  for (int i = 1; i < N; ++i) {
    if (!THPVariable_Check(args[i])) continue;
    const at::Tensor &t = THPVariable_Unpack(args[i]);
    if (t.is_cuda() && t.device() != first) {
      PyErr_Format(PyExc_ValueError, "%s: on %s, %s on %s", ops[i].name, t.device().str().c_str(), ops[0].name, first.str().c_str());
      return false;
    }
  }
  const int current = c10::hip::current_device();
  if (first.index() != current) {
    PyErr_Format(PyExc_ValueError, "%s: on %s, the current device is cuda:%d", ops[0].name, first.str().c_str(), current);
    return false;
  }
  return true;
}
template <int N>
bool describe_all(PyObject *const *args, const Operand (&ops)[N], npu_memref (&m)[N]) {
  if (!on_current_device(args, ops)) return false;
  for (int i = 0; i < N; ++i)
    if (!describe(args[i], ops[i].name, ops[i].optional, &m[i])) return false;
  return true;
}

bool counted(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", n, want);
  return false;
}

bool int32_of(PyObject *o, const char *name, int32_t *v) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) return false;
  if (x != (int32_t)x) {
    PyErr_Format(PyExc_ValueError, "%s: %lld is no 32-bit integer", name, x);
    return false;
  }
  *v = (int32_t)x;
  return true;
}

// A raw handle, or None: torch's current stream.
bool stream_of(PyObject *o, npu_stream *s) {
  *s = o == Py_None ? c10::hip::getCurrentHIPStream().stream() : PyLong_AsVoidPtr(o);
  return !PyErr_Occurred();
}

// Each returns the entry point's status; C++ exceptions (a tensor without
// storage) become Python errors.
template <class F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject *rope_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[11] = {{"Q", false}, {"K", false}, {"V", false}, {"cos_t", false}, {"sin_t", false},
                                  {"k_pages", false}, {"v_pages", false}, {"page_table", false}, {"kv_len", false},
                                  {"q_start", true}, {"Qo", false}};
  return guarded([&]() -> PyObject * {
    npu_memref m[11];
    int32_t prefix_len, pairs;
    npu_stream s;
    if (!counted(n, 14) || !describe_all(a, ops, m) || !int32_of(a[11], "prefix_len", &prefix_len) ||
        !int32_of(a[12], "pairs", &pairs) || !stream_of(a[13], &s))
      return nullptr;
    return PyLong_FromLong(fused_llama_rope_append(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], &m[6], &m[7], &m[8],
                                                   &m[9], &m[10], prefix_len, pairs, s));
  });
}

PyObject *paged_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[9] = {{"Q", false}, {"k_pages", false}, {"v_pages", false}, {"page_table", false},
                                 {"kv_len", false}, {"q_start", true}, {"prefix_table", true}, {"A", false},
                                 {"workspace", false}};
  return guarded([&]() -> PyObject * {
    npu_memref m[9];
    int32_t prefix_len;
    npu_stream s;
    if (!counted(n, 12) || !describe_all(a, ops, m) || !int32_of(a[9], "prefix_len", &prefix_len)) return nullptr;
    const double scale = PyFloat_AsDouble(a[10]);
    if (PyErr_Occurred() || !stream_of(a[11], &s)) return nullptr;
    return PyLong_FromLong(fused_llama_paged_attention(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], &m[6], &m[7], &m[8],
                                                       prefix_len, (float)scale, s));
  });
}

PyObject *sample_tokens(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[9] = {{"logits", false}, {"u", false}, {"temperature", true}, {"top_k", true},
                                 {"top_p", true}, {"min_p", true}, {"tokens", false}, {"probs", true},
                                 {"workspace", false}};
  return guarded([&]() -> PyObject * {
    npu_memref m[9];
    npu_stream s;
    if (!counted(n, 10) || !describe_all(a, ops, m) || !stream_of(a[9], &s)) return nullptr;
    return PyLong_FromLong(fused_sample_tokens(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], &m[6], &m[7], &m[8], s));
  });
}

PyObject *token_logprobs(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[8] = {{"logits", false}, {"tokens", false}, {"logprobs", false}, {"entropy", true},
                                 {"ranks", true}, {"top_tokens", true}, {"top_logprobs", true}, {"workspace", false}};
  return guarded([&]() -> PyObject * {
    npu_memref m[8];
    npu_stream s;
    if (!counted(n, 9) || !describe_all(a, ops, m) || !stream_of(a[8], &s)) return nullptr;
    return PyLong_FromLong(fused_token_logprobs(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], &m[6], &m[7], s));
  });
}

PyObject *mx_quantize(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[5] = {{"x", false}, {"gate", true}, {"q", false}, {"scale", false}, {"values", true}};
  return guarded([&]() -> PyObject * {
    npu_memref m[5];
    npu_stream s;
    if (!counted(n, 6) || !describe_all(a, ops, m) || !stream_of(a[5], &s)) return nullptr;
    return PyLong_FromLong(fused_mx_quantize(&m[0], &m[1], &m[2], &m[3], &m[4], s));
  });
}

PyObject *add_rmsnorm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[6] = {{"x", false}, {"delta", true}, {"g", false}, {"h", true}, {"q", false}, {"scale", true}};
  return guarded([&]() -> PyObject * {
    npu_memref m[6];
    npu_stream s;
    if (!counted(n, 8) || !describe_all(a, ops, m)) return nullptr;
    const double eps = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred() || !stream_of(a[7], &s)) return nullptr;
    return PyLong_FromLong(fused_llama_add_rmsnorm(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], (float)eps, s));
  });
}

PyObject *mx_matmul(PyObject *, PyObject *const *a, Py_ssize_t n) {
  static const Operand ops[6] = {{"a", false}, {"a_scale", false}, {"w", false}, {"w_scale", false}, {"out", false},
                                 {"workspace", false}};
  return guarded([&]() -> PyObject * {
    npu_memref m[6];
    npu_stream s;
    if (!counted(n, 7) || !describe_all(a, ops, m) || !stream_of(a[6], &s)) return nullptr;
    return PyLong_FromLong(fused_mx_matmul(&m[0], &m[1], &m[2], &m[3], &m[4], &m[5], s));
  });
}

PyMethodDef methods[] = {
    {"rope_append", (PyCFunction)(void (*)(void))rope_append, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {"sample_tokens", (PyCFunction)(void (*)(void))sample_tokens, METH_FASTCALL, nullptr},
    {"token_logprobs", (PyCFunction)(void (*)(void))token_logprobs, METH_FASTCALL, nullptr},
    {"mx_quantize", (PyCFunction)(void (*)(void))mx_quantize, METH_FASTCALL, nullptr},
    {"add_rmsnorm", (PyCFunction)(void (*)(void))add_rmsnorm, METH_FASTCALL, nullptr},
    {"mx_matmul", (PyCFunction)(void (*)(void))mx_matmul, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve(void) { return PyModule_Create(&module); }
