// Python binding of the token-decoding operators (ops.qkv_rope_append, kv4_read, kv4_attention, sample):
// checks the tensors, allocates the results and calls the C ABI on the current stream.
//
// A decode step makes a few launches of some microseconds per layer, so what the host spends on a call
// counts: the same steps through ctypes took 14 us a call, of which the launch is 3.  The C ABI's entry
// points and the error class are handed over by bind(), so the process has one librldx_b200.so.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/rldx_b200.h"

namespace {

decltype(&rldx_last_error) g_last_error = nullptr;
decltype(&rldx_kv4_append) g_append = nullptr;
decltype(&rldx_kv4_read) g_read = nullptr;
decltype(&rldx_kv4_attention_workspace_size) g_workspace = nullptr;
decltype(&rldx_kv4_attention) g_attention = nullptr;
decltype(&rldx_sample) g_sample = nullptr;
PyObject* g_error = nullptr;

// A refusal: TypeError or ValueError with a message.
struct Refused {
  PyObject* type;
  std::string msg;
};
[[noreturn]] void refuse_value(const std::string& msg) { throw Refused{PyExc_ValueError, msg}; }
[[noreturn]] void refuse_type(const std::string& msg) { throw Refused{PyExc_TypeError, msg}; }
// A Python error is set already.
struct Raised {};

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse_type(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
int small(PyObject* o, const char* name) {
  const long v = integer(o);
  if (v != static_cast<int>(v)) refuse_value(std::string(name) + " does not fit 32 bits");
  return static_cast<int>(v);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

void check(int rc) {
  if (rc == RLDX_OK) return;
  PyObject* e = PyObject_CallFunction(g_error, "is", rc, g_last_error());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Raised{};
}

// The device that holds every tensor; it has to be the current one, whose stream the launch goes to.
class Device {
 public:
  explicit Device(const at::Tensor& t) : index_(t.is_cuda() ? t.get_device() : -1) {
    if (index_ < 0 || index_ != c10::cuda::current_device())
      refuse_value("every tensor must be on the current CUDA device, got " + t.device().str() + " (no CPU path exists)");
  }
  void has(const at::Tensor& t) const {
    if (!t.is_cuda() || t.get_device() != index_)
      refuse_value("the tensors are on different devices: cuda:" + std::to_string(index_) + " and " + t.device().str());
  }
  void has(const at::Tensor* t) const {
    if (t) has(*t);
  }
  at::Tensor empty(at::IntArrayRef size, at::ScalarType type) const {
    return at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(index_)), std::nullopt);
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index_)).stream(); }

 private:
  int64_t index_;
};

void vector_of(const at::Tensor& t, const char* name, at::ScalarType type, const char* type_name, int64_t n) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
    refuse_value(std::string(name) + " must be a contiguous " + type_name + " tensor [" + std::to_string(n) + "]");
}

rldx_kv4_cache cache_of(const Device& dev, PyObject* const* a) {  // cache, table, lengths, cu_seqlens
  const at::Tensor &cache = tensor(a[0], "cache"), &table = tensor(a[1], "table"), &lengths = tensor(a[2], "lengths"),
                   &cu = tensor(a[3], "cu_seqlens");
  dev.has(cache), dev.has(table), dev.has(lengths), dev.has(cu);
  if (cache.scalar_type() != at::kByte || cache.dim() != 4 || !cache.is_contiguous() ||
      (cache.size(3) != 2560 && cache.size(3) != 5120))
    refuse_value("cache must be a contiguous uint8 tensor [pages, kv_heads, page_size / 32, 40 head_dim], head_dim 64 or 128");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.stride(1) != 1)
    refuse_value("table must be a row-major int32 tensor [seqs, pages of a sequence]");
  const int64_t seqs = table.size(0), width = table.size(1);
  vector_of(lengths, "lengths", at::kInt, "int32", seqs);
  vector_of(cu, "cu_seqlens", at::kInt, "int32", seqs + 1);
  if (width > INT32_MAX || seqs > INT32_MAX || cache.size(1) > INT32_MAX || cache.size(2) > INT32_MAX / 32)
    refuse_value("a dimension of the cache or the table does not fit 32 bits");
  const int64_t ld = seqs > 1 ? table.stride(0) : width;
  if (ld > INT32_MAX) refuse_value("the table's row stride does not fit 32 bits");
  rldx_kv4_cache c;
  c.data = cache.mutable_data_ptr();
  c.table = static_cast<const int32_t*>(table.const_data_ptr());
  c.lengths = static_cast<const int32_t*>(lengths.const_data_ptr());
  c.cu_seqlens = static_cast<const int32_t*>(cu.const_data_ptr());
  c.pages = cache.size(0);
  c.page_size = static_cast<int>(32 * cache.size(2));
  c.kv_heads = static_cast<int>(cache.size(1));
  c.head_dim = static_cast<int>(cache.size(3) / 40);
  c.table_width = static_cast<int>(width);
  c.table_ld = static_cast<int>(ld);
  c.seqs = static_cast<int>(seqs);
  return c;
}

int rows_of(int64_t n) {
  if (n > INT32_MAX) refuse_value("more than 2^31 rows");
  return static_cast<int>(n);
}

bool side_by_side(const at::Tensor& t, int64_t rows, int64_t heads, int64_t d) {
  return t.scalar_type() == at::kBFloat16 && t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == d &&
         t.is_contiguous();
}

template <typename F>
PyObject* guarded(const char* name, Py_ssize_t got, Py_ssize_t want, F f) {
  HANDLE_TH_ERRORS
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, got);
    return nullptr;
  }
  if (!g_error) {
    PyErr_SetString(PyExc_RuntimeError, "the binding is not bound to the library");
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.msg.c_str());
  } catch (const Raised&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

// qkv, q_norm, k_norm, cos, sin, rope_pos, cache, table, lengths, cu_seqlens, q_heads, eps, out
PyObject* qkv_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("qkv_rope_append", n, 13, [&] {
    const at::Tensor &qkv = tensor(a[0], "qkv"), &qn = tensor(a[1], "q_norm"), &kn = tensor(a[2], "k_norm"),
                     &cos = tensor(a[3], "cos"), &sin = tensor(a[4], "sin"), &pos = tensor(a[5], "rope_pos");
    const at::Tensor* out = optional_tensor(a[12], "out");
    const auto bf = at::kBFloat16;
    if (qkv.scalar_type() != bf || qn.scalar_type() != bf || kn.scalar_type() != bf || pos.scalar_type() != at::kInt)
      refuse_type("qkv, q_norm and k_norm must be bfloat16, rope_pos int32");
    const bool fp32 = cos.scalar_type() == at::kFloat;
    if ((!fp32 && cos.scalar_type() != bf) || sin.scalar_type() != cos.scalar_type())
      refuse_type("cos and sin must both be bfloat16 or both float32");
    const Device dev(qkv);
    dev.has(qn), dev.has(kn), dev.has(cos), dev.has(sin), dev.has(pos), dev.has(out);
    const rldx_kv4_cache c = cache_of(dev, a + 6);
    const int q_heads = small(a[10], "q_heads");
    const int64_t d = c.head_dim, width = (static_cast<int64_t>(q_heads) + 2 * c.kv_heads) * d;
    if (qkv.dim() != 2 || qkv.stride(1) != 1) refuse_value("qkv must be a 2-D row-major view");
    if (qkv.size(1) != width)
      refuse_value("qkv rows must hold (q_heads + 2 kv_heads) head_dim = " + std::to_string(width) + " values, got " +
                   std::to_string(qkv.size(1)));
    const int tokens = rows_of(qkv.size(0));
    if (qn.dim() != 1 || qn.size(0) != d || !qn.is_contiguous() || kn.dim() != 1 || kn.size(0) != d || !kn.is_contiguous())
      refuse_value("q_norm and k_norm must be contiguous [" + std::to_string(d) + "]");
    if (cos.dim() != 2 || cos.size(1) != d || !cos.is_contiguous() || sin.sizes() != cos.sizes() || !sin.is_contiguous())
      refuse_value("cos and sin must be contiguous [rows, " + std::to_string(d) + "]");
    vector_of(pos, "rope_pos", at::kInt, "int32", tokens);
    if (out && !side_by_side(*out, tokens, q_heads, d))
      refuse_value("out must be a contiguous bfloat16 tensor [" + std::to_string(tokens) + ", " + std::to_string(q_heads) + ", " +
                   std::to_string(d) + "]");
    const at::Tensor q = out ? *out : dev.empty({tokens, q_heads, d}, bf);
    if (tokens > 0)
      check(g_append(&c, qkv.const_data_ptr(), tokens > 1 ? qkv.stride(0) : width, tokens, q_heads,
                     qn.const_data_ptr(), kn.const_data_ptr(), cos.const_data_ptr(), sin.const_data_ptr(), fp32,
                     rows_of(cos.size(0)), static_cast<const int32_t*>(pos.const_data_ptr()), q.mutable_data_ptr(),
                     static_cast<float>(number(a[11])), dev.stream()));
    return THPVariable_Wrap(q);
  });
}

// cache, table, lengths, cu_seqlens, tokens
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("kv4_read", n, 5, [&] {
    const Device dev(tensor(a[0], "cache"));
    const rldx_kv4_cache c = cache_of(dev, a);
    const int tokens = small(a[4], "tokens");
    if (tokens < 0) refuse_value("tokens must not be negative");
    const at::Tensor k = dev.empty({tokens, c.kv_heads, c.head_dim}, at::kBFloat16), v = dev.empty(k.sizes(), at::kBFloat16);
    if (tokens > 0) check(g_read(&c, tokens, k.mutable_data_ptr(), v.mutable_data_ptr(), dev.stream()));
    PyObject* both = PyTuple_New(2);
    if (!both) throw Raised{};
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(k));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(v));
    return both;
  });
}

// q, cache, table, lengths, cu_seqlens, max_new, max_len, window, sinks, scale, out
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("kv4_attention", n, 11, [&] {
    const at::Tensor& q = tensor(a[0], "q");
    const at::Tensor* out = optional_tensor(a[10], "out");
    if (q.scalar_type() != at::kBFloat16) refuse_type("q must be bfloat16");
    const Device dev(q);
    dev.has(out);
    const rldx_kv4_cache c = cache_of(dev, a + 1);
    const int64_t d = c.head_dim;
    if (q.dim() != 3 || q.size(2) != d || q.stride(2) != 1 || (q.size(1) > 1 && q.stride(1) != d))
      refuse_value("q must be [tokens, q_heads, " + std::to_string(d) + "] with the heads of a token side by side");
    rldx_kv4_attention_desc t;
    t.tokens = rows_of(q.size(0));
    t.q_heads = rows_of(q.size(1));
    if (out && !side_by_side(*out, q.size(0), q.size(1), d))
      refuse_value("out must be a contiguous bfloat16 tensor of q's shape");
    const at::Tensor o = out ? *out : dev.empty({q.size(0), q.size(1), d}, at::kBFloat16);
    t.q = q.const_data_ptr();
    t.out = o.mutable_data_ptr();
    t.ldq = t.tokens > 1 ? q.stride(0) : q.size(1) * d;
    t.max_new = small(a[5], "max_new");
    t.max_len = small(a[6], "max_len");
    t.window = small(a[7], "window");
    t.sinks = small(a[8], "sinks");
    t.scale = a[9] == Py_None ? 1.0f / std::sqrt(static_cast<float>(d)) : static_cast<float>(number(a[9]));
    if (t.tokens > 0) {
      uint64_t bytes = 0;
      check(g_workspace(&c, &t, &bytes));
      at::Tensor ws;
      if (bytes) ws = dev.empty({static_cast<int64_t>(bytes)}, at::kByte);
      check(g_attention(&c, &t, bytes ? ws.mutable_data_ptr() : nullptr, bytes, dev.stream()));
    }
    return THPVariable_Wrap(o);
  });
}

// logits, u, temperature, top_k, top_p, min_p
PyObject* sample(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("sample", n, 6, [&] {
    const at::Tensor &logits = tensor(a[0], "logits"), &u = tensor(a[1], "u");
    const bool fp32 = logits.scalar_type() == at::kFloat;
    if (!fp32 && logits.scalar_type() != at::kBFloat16) refuse_type("logits must be bfloat16 or float32");
    const Device dev(logits);
    dev.has(u);
    if (logits.dim() != 2 || logits.stride(1) != 1) refuse_value("logits must be a 2-D row-major view");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    vector_of(u, "u", at::kFloat, "float32", rows);
    static const char* const names[4] = {"temperature", "top_k", "top_p", "min_p"};
    const void* limit[4];
    for (int i = 0; i < 4; ++i) {
      const at::Tensor* t = optional_tensor(a[2 + i], names[i]);
      limit[i] = nullptr;
      if (!t) continue;
      dev.has(t);
      vector_of(*t, names[i], i == 1 ? at::kInt : at::kFloat, i == 1 ? "int32" : "float32", rows);
      limit[i] = t->const_data_ptr();
    }
    const at::Tensor token = dev.empty({rows}, at::kLong), logprob = dev.empty({rows}, at::kFloat), kept = dev.empty({rows}, at::kInt);
    if (rows > 0)
      check(g_sample(logits.const_data_ptr(), rows > 1 ? logits.stride(0) : vocab, rows_of(rows),
                     rows_of(vocab), fp32, static_cast<const float*>(u.const_data_ptr()), static_cast<const float*>(limit[0]),
                     static_cast<const int32_t*>(limit[1]), static_cast<const float*>(limit[2]), static_cast<const float*>(limit[3]),
                     static_cast<int64_t*>(token.mutable_data_ptr()), static_cast<float*>(logprob.mutable_data_ptr()),
                     static_cast<int32_t*>(kept.mutable_data_ptr()), dev.stream()));
    PyObject* all = PyTuple_New(3);
    if (!all) throw Raised{};
    PyTuple_SET_ITEM(all, 0, THPVariable_Wrap(token));
    PyTuple_SET_ITEM(all, 1, THPVariable_Wrap(logprob));
    PyTuple_SET_ITEM(all, 2, THPVariable_Wrap(kept));
    return all;
  });
}

// error class, then the addresses of the entry points in the order of the globals above
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind takes the error class and six addresses");
    return nullptr;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[1 + i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  }
  g_last_error = reinterpret_cast<decltype(g_last_error)>(p[0]);
  g_append = reinterpret_cast<decltype(g_append)>(p[1]);
  g_read = reinterpret_cast<decltype(g_read)>(p[2]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[3]);
  g_attention = reinterpret_cast<decltype(g_attention)>(p[4]);
  g_sample = reinterpret_cast<decltype(g_sample)>(p[5]);
  Py_INCREF(a[0]);
  Py_XDECREF(g_error);
  g_error = a[0];
  Py_RETURN_NONE;
}

#define RLDX_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {RLDX_METHOD(bind),          RLDX_METHOD(qkv_rope_append), RLDX_METHOD(kv4_read),
                           RLDX_METHOD(kv4_attention), RLDX_METHOD(sample),          {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&g_module); }
