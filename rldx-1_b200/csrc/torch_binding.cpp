// Python binding of the token-decoding operators (ops.qkv_rope_append, kv4_read, kv4_attention, sample, rope,
// rope_rows, block_norms, token_logprobs): checks the tensors, allocates the results and calls the C ABI on the
// current stream.
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
decltype(&rldx_rope) g_rope = nullptr;
decltype(&rldx_rope_rows) g_rope_rows = nullptr;
decltype(&rldx_block_norms) g_block_norms = nullptr;
decltype(&rldx_token_logprobs) g_token_logprobs = nullptr;
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

int small_count(int64_t n, const char* name) {
  if (n > INT32_MAX) refuse_value(std::string(name) + " does not fit 32 bits");
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

// ---- rotary positions, block norms, log probabilities ----
// These look at shapes, types and layouts before the device, so a wrong call is refused alike on every machine.

int dtype_of(at::ScalarType t, const char* name) {
  if (t == at::kBFloat16) return RLDX_BF16;
  if (t == at::kHalf) return RLDX_F16;
  if (t == at::kFloat) return RLDX_F32;
  refuse_type(std::string(name) + " must be bfloat16, float16 or float32");
}

// Whether a tensor of rows (dimension 0; the others densely or in steps below the rows') is apart from another: no byte
// of one between the first and last of the other, or both of one row stride and in columns of their own.
struct Span {
  uintptr_t first;
  int64_t rows, stride, width, size;  // elements, and bytes of one
  explicit Span(const at::Tensor& t) : first(reinterpret_cast<uintptr_t>(t.const_data_ptr())), rows(t.size(0)), stride(t.stride(0)), width(1), size(t.element_size()) {
    for (int64_t i = 1; i < t.dim(); ++i) width += (t.size(i) - 1) * t.stride(i);
    if (t.numel() == 0) rows = 0;
  }
  uintptr_t end() const { return rows ? first + ((rows - 1) * stride + width) * size : first; }
  bool apart_from(const Span& o) const {
    if (!rows || !o.rows || end() <= o.first || o.end() <= first) return true;
    const int64_t row = stride * size, d = static_cast<int64_t>(o.first - first);
    if (row <= 0 || row != o.stride * o.size || width * size > row || o.width * o.size > row) return false;
    const int64_t column = ((d % row) + row) % row;  // where o's rows begin in this one's
    return column >= width * size && column + o.width * o.size <= row;
  }
};
bool same_place(const at::Tensor& a, const at::Tensor& b) {
  return a.const_data_ptr() == b.const_data_ptr() && a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes() && a.strides() == b.strides();
}
// A written tensor may be one of what is read, place for place, and has to be apart from the rest.
void writes_apart(const at::Tensor& out, const char* name, const at::Tensor* in, const char* in_name) {
  if (in && !same_place(out, *in) && !Span(out).apart_from(Span(*in)))
    refuse_value(std::string(name) + " shares memory with " + in_name + ": it may be the same tensor, or one apart from it");
}

// positions, freqs, sections, interleaved_sections, interleaved, factor, inverse
struct RopePlan {
  const at::Tensor *positions, *freqs;
  int64_t tokens;
  rldx_rope_plan p = {};
  explicit RopePlan(PyObject* const* a) : positions(&tensor(a[0], "positions")), freqs(&tensor(a[1], "freqs")) {
    if (positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong) refuse_type("positions must be int32 or int64");
    if (freqs->scalar_type() != at::kDouble) refuse_type("freqs must be float64");
    if (freqs->dim() != 1 || freqs->size(0) < 1 || !freqs->is_contiguous()) refuse_value("freqs must be a contiguous tensor [pairs]");
    if (freqs->size(0) > 512) refuse_value("freqs must be of at most 512 pairs");
    p.pairs = static_cast<int>(freqs->size(0));
    p.axes = 1;
    if (a[2] != Py_None) {
      PyObject* seq = PySequence_Fast(a[2], "sections must be a sequence of whole numbers");
      if (!seq) throw Raised{};
      const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
      long v[4] = {0, 0, 0, 0}, sum = 0;
      for (Py_ssize_t i = 0; i < n && i < 4; ++i) {
        v[i] = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
        if (v[i] == -1 && PyErr_Occurred()) {
          Py_DECREF(seq);
          throw Raised{};
        }
      }
      Py_DECREF(seq);
      if (n < 1 || n > 4) refuse_value("sections must be of 1 to 4 axes");
      for (int i = 0; i < n; ++i) {
        if (v[i] < 0 || v[i] > p.pairs) refuse_value("sections must be counts of pairs");
        p.sections[i] = static_cast<int>(v[i]);
        sum += v[i];
      }
      if (sum != p.pairs) refuse_value("sections must add up to the " + std::to_string(p.pairs) + " pairs of freqs");
      p.axes = static_cast<int>(n);
    }
    const int64_t dim = positions->dim();
    if (dim != 1 && dim != 2) refuse_value("positions must be [tokens] or [axes, tokens]");
    if (dim == 1 ? p.axes != 1 : positions->size(0) != p.axes)
      refuse_value("positions must have " + std::to_string(p.axes) + " axes, as sections say");
    tokens = positions->size(dim - 1);
    if (tokens > 1 && positions->stride(dim - 1) != 1) refuse_value("positions of an axis must lie side by side");
    p.positions_ld = dim == 2 ? positions->stride(0) : 0;
    p.positions_int64 = positions->scalar_type() == at::kLong;
    p.sections_interleaved = truth(a[3]);
    p.interleaved = truth(a[4]);
    p.factor = static_cast<float>(number(a[5]));
    p.inverse = truth(a[6]);
  }
  static int truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v;
  }
  void at(const Device& dev) {
    dev.has(*positions), dev.has(*freqs);
    p.positions = positions->const_data_ptr();
    p.freqs = static_cast<const double*>(freqs->const_data_ptr());
  }
};

// q, k, positions, freqs, sections, interleaved_sections, interleaved, factor, inverse, out_q, out_k
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("rope", n, 11, [&] {
    static const char* const names[2] = {"q", "k"};
    static const char* const out_names[2] = {"out_q", "out_k"};
    const at::Tensor* x[2] = {&tensor(a[0], "q"), optional_tensor(a[1], "k")};
    const at::Tensor* given[2] = {optional_tensor(a[9], "out_q"), optional_tensor(a[10], "out_k")};
    RopePlan plan(a + 2);
    const int dtype = dtype_of(x[0]->scalar_type(), "q");
    if (given[1] && !x[1]) refuse_value("out_k goes with k");
    for (int i = 0; i < 2; ++i) {
      if (!x[i]) continue;
      const at::Tensor& t = *x[i];
      if (t.scalar_type() != x[0]->scalar_type()) refuse_type("q and k must have one type");
      if (t.dim() != 3 || t.size(0) != plan.tokens || t.size(2) != x[0]->size(2) || t.stride(2) != 1)
        refuse_value(std::string(names[i]) + " must be [" + std::to_string(plan.tokens) + " tokens, heads, head_dim] with a head's values side by side");
      if (t.size(1) < 1) refuse_value(std::string(names[i]) + " has no heads");
      if (t.size(2) < 2 * plan.p.pairs)
        refuse_value("a head of " + std::to_string(t.size(2)) + " values has no " + std::to_string(plan.p.pairs) + " pairs");
      if (given[i]) {
        if (given[i]->scalar_type() != t.scalar_type()) refuse_type(std::string(out_names[i]) + " must have q's type");
        if (given[i]->sizes() != t.sizes() || given[i]->stride(2) != 1)
          refuse_value(std::string(out_names[i]) + " must have the shape of what it takes, a head's values side by side");
        writes_apart(*given[i], out_names[i], x[i], names[i]);
        if (x[1 - i] && !Span(*given[i]).apart_from(Span(*x[1 - i])))
          refuse_value(std::string(out_names[i]) + " shares memory with " + names[1 - i]);
        for (const at::Tensor* t : {plan.positions, plan.freqs})  // (other blocks read them still)
          if (!Span(*given[i]).apart_from(Span(*t)))
            refuse_value(std::string(out_names[i]) + " shares memory with " + (t == plan.freqs ? "freqs" : "positions"));
      }
    }
    if (given[0] && given[1] && !Span(*given[0]).apart_from(Span(*given[1]))) refuse_value("out_q and out_k share memory");
    const Device dev(*x[0]);
    dev.has(x[1]), dev.has(given[0]), dev.has(given[1]);
    plan.at(dev);
    at::Tensor out[2];
    rldx_rope_heads h[2];
    int parts = 0;
    for (int i = 0; i < 2; ++i) {
      if (!x[i]) continue;
      const at::Tensor& t = *x[i];
      out[i] = given[i] ? *given[i] : dev.empty(t.sizes(), t.scalar_type());
      if (plan.tokens == 0) continue;
      const bool one = plan.tokens == 1, single = t.size(1) == 1;
      h[parts++] = {t.const_data_ptr(), out[i].mutable_data_ptr(), one ? 0 : t.stride(0), single ? 0 : t.stride(1),
                    one ? 0 : out[i].stride(0), single ? 0 : out[i].stride(1), small_count(t.size(1), "heads")};
    }
    if (plan.tokens > 0) check(g_rope(&plan.p, h, parts, plan.tokens, small_count(x[0]->size(2), "head_dim"), dtype, dev.stream()));
    PyObject* both = PyTuple_New(2);
    if (!both) throw Raised{};
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(out[0]));
    if (x[1]) {
      PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(out[1]));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(both, 1, Py_None);
    }
    return both;
  });
}

// positions, freqs, sections, interleaved_sections, factor, inverse, type (RLDX_BF16, ...)
PyObject* rope_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("rope_rows", n, 7, [&] {
    PyObject* const whole[7] = {a[0], a[1], a[2], a[3], Py_False, a[4], a[5]};
    RopePlan plan(whole);
    const int dtype = small(a[6], "dtype");
    const at::ScalarType type = dtype == RLDX_BF16 ? at::kBFloat16 : dtype == RLDX_F16 ? at::kHalf : at::kFloat;
    const Device dev(*plan.positions);
    plan.at(dev);
    const at::Tensor cos = dev.empty({plan.tokens, 2 * plan.p.pairs}, type), sin = dev.empty(cos.sizes(), type);
    if (plan.tokens > 0) check(g_rope_rows(&plan.p, plan.tokens, cos.mutable_data_ptr(), sin.mutable_data_ptr(), dtype, dev.stream()));
    PyObject* both = PyTuple_New(2);
    if (!both) throw Raised{};
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(cos));
    PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(sin));
    return both;
  });
}

// branch, residual, post, post_weight, post_bias, gate, scale, pre, pre_weight, pre_bias, mod_scale, mod_shift,
// rows_per_group, weight_plus_one, eps, out_residual, out
PyObject* block_norms(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("block_norms", n, 17, [&] {
    const at::Tensor &y = tensor(a[0], "branch"), &h = tensor(a[1], "residual");
    rldx_block_norms_desc d = {};
    d.dtype = dtype_of(y.scalar_type(), "branch");
    d.residual_dtype = dtype_of(h.scalar_type(), "residual");
    if (d.residual_dtype != d.dtype && d.residual_dtype != RLDX_F32) refuse_type("residual must have branch's type or float32");
    if (y.dim() != 2 || (y.size(1) > 1 && y.stride(1) != 1)) refuse_value("branch must be a 2-D row-major view");
    const int64_t rows = y.size(0), width = y.size(1);
    if (h.sizes() != y.sizes() || (width > 1 && h.stride(1) != 1)) refuse_value("residual must be a row-major view of branch's shape");
    if (width < 1 || width > 14336) refuse_value("rows must have 1 to 14336 values");
    d.post = small(a[2], "post"), d.pre = small(a[7], "pre");
    d.rows = rows, d.width = static_cast<int>(width);
    d.rows_per_group = integer(a[12]);
    if (d.rows_per_group < 0) refuse_value("rows_per_group must not be negative");
    d.scale = static_cast<float>(number(a[6])), d.eps = static_cast<float>(number(a[14]));
    d.weight_plus_one = RopePlan::truth(a[13]);
    const int at[7] = {3, 4, 5, 8, 9, 10, 11};
    static const char* const names[7] = {"post_weight", "post_bias", "gate", "pre_weight", "pre_bias", "mod_scale", "mod_shift"};
    const void** to[7] = {&d.post_weight, &d.post_bias, &d.gate, &d.pre_weight, &d.pre_bias, &d.mod_scale, &d.mod_shift};
    int64_t* ld[7] = {nullptr, nullptr, &d.ld_gate, nullptr, nullptr, &d.ld_scale, &d.ld_shift};
    const at::Tensor* vec[7];
    const at::Tensor* first = nullptr;
    d.vector_dtype = d.dtype;
    for (int i = 0; i < 7; ++i) {
      vec[i] = optional_tensor(a[at[i]], names[i]);
      if (!vec[i]) continue;
      const at::Tensor& v = *vec[i];
      const int type = dtype_of(v.scalar_type(), names[i]);
      if (!first) first = vec[i], d.vector_dtype = type;
      if (type != d.vector_dtype || (type != d.dtype && type != RLDX_F32))
        refuse_type("weights, biases, gate and modulation must all have branch's type, or all float32");
      const bool groups = ld[i] && v.dim() == 2;
      if (!groups && (v.dim() != 1 || v.size(0) != width || (width > 1 && v.stride(0) != 1)))
        refuse_value(std::string(names[i]) + " must be a contiguous tensor [" + std::to_string(width) + "]" + (ld[i] ? " or row-major [groups, ...]" : ""));
      if (groups) {
        if (v.size(1) != width || (width > 1 && v.stride(1) != 1))
          refuse_value(std::string(names[i]) + " must be row-major [groups, " + std::to_string(width) + "]");
        if (d.rows_per_group < 1) refuse_value(std::string(names[i]) + " of groups needs rows_per_group");
        if (v.size(0) != (rows > 0 ? 1 + (rows - 1) / d.rows_per_group : 0))
          refuse_value(std::string(names[i]) + " must have a row for each group of " + std::to_string(d.rows_per_group) + " rows");
        *ld[i] = v.size(0) > 1 ? v.stride(0) : 0;
      }
    }
    const at::Tensor *given_h = optional_tensor(a[15], "out_residual"), *given_n = optional_tensor(a[16], "out");
    if (given_n && d.pre == RLDX_NORM_NONE) refuse_value("without a pre norm there is no out");
    for (int i = 0; i < 2; ++i) {
      const at::Tensor* t = i ? given_n : given_h;
      const char* name = i ? "out" : "out_residual";
      if (!t) continue;
      if (t->scalar_type() != (i ? y : h).scalar_type()) refuse_type(std::string(name) + " must have the type of " + (i ? "branch" : "residual"));
      if (t->sizes() != y.sizes() || (width > 1 && t->stride(1) != 1) || (rows > 1 && t->stride(0) < width))
        refuse_value(std::string(name) + " must be a row-major view of branch's shape");
      writes_apart(*t, name, &y, "branch");
      writes_apart(*t, name, &h, "residual");
      for (int v = 0; v < 7; ++v)
        if (vec[v] && !Span(*t).apart_from(Span(vec[v]->dim() == 1 ? vec[v]->unsqueeze(0) : *vec[v]))) refuse_value(std::string(name) + " shares memory with " + names[v]);
    }
    if (given_h && given_n && !Span(*given_h).apart_from(Span(*given_n))) refuse_value("out_residual and out share memory");
    const Device dev(y);
    dev.has(h), dev.has(given_h), dev.has(given_n);
    for (int i = 0; i < 7; ++i) {
      dev.has(vec[i]);
      if (vec[i]) *to[i] = vec[i]->const_data_ptr();
    }
    const at::Tensor h_out = given_h ? *given_h : dev.empty(y.sizes(), h.scalar_type());
    at::Tensor n_out;
    if (d.pre != RLDX_NORM_NONE) n_out = given_n ? *given_n : dev.empty(y.sizes(), y.scalar_type());
    d.branch = y.const_data_ptr(), d.residual = h.const_data_ptr(), d.residual_out = h_out.mutable_data_ptr();
    if (n_out.defined()) d.out = n_out.mutable_data_ptr();
    auto stride = [&](const at::Tensor& t) { return rows > 1 ? t.stride(0) : width; };
    d.ld_branch = stride(y), d.ld_residual = stride(h), d.ld_residual_out = stride(h_out), d.ld_out = n_out.defined() ? stride(n_out) : 0;
    if (rows > 0) check(g_block_norms(&d, dev.stream()));
    PyObject* both = PyTuple_New(2);
    if (!both) throw Raised{};
    PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(h_out));
    if (n_out.defined()) {
      PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(n_out));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(both, 1, Py_None);
    }
    return both;
  });
}

// logits, tokens, top
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded("token_logprobs", n, 3, [&] {
    const at::Tensor &logits = tensor(a[0], "logits"), &tokens = tensor(a[1], "tokens");
    const int dtype = dtype_of(logits.scalar_type(), "logits");
    if (logits.dim() != 2 || (logits.size(1) > 1 && logits.stride(1) != 1)) refuse_value("logits must be a 2-D row-major view");
    const int64_t rows = logits.size(0), vocab = logits.size(1);
    if (vocab < 1) refuse_value("logits have no tokens");
    vector_of(tokens, "tokens", at::kLong, "int64", rows);
    const int top = small(a[2], "top");
    if (top < 0 || top > 32 || top > vocab) refuse_value("top must be 0 to 32, and no more than the tokens");
    const Device dev(logits);
    dev.has(tokens);
    const at::Tensor logprob = dev.empty({rows}, at::kFloat), entropy = dev.empty({rows}, at::kFloat), rank = dev.empty({rows}, at::kInt),
                     ids = dev.empty({rows, top}, at::kLong), values = dev.empty({rows, top}, at::kFloat);
    if (rows > 0)
      check(g_token_logprobs(logits.const_data_ptr(), rows > 1 ? logits.stride(0) : vocab, rows_of(rows), rows_of(vocab), dtype,
                             static_cast<const int64_t*>(tokens.const_data_ptr()), top, static_cast<float*>(logprob.mutable_data_ptr()),
                             static_cast<float*>(entropy.mutable_data_ptr()), static_cast<int32_t*>(rank.mutable_data_ptr()),
                             top ? static_cast<int64_t*>(ids.mutable_data_ptr()) : nullptr,
                             top ? static_cast<float*>(values.mutable_data_ptr()) : nullptr, dev.stream()));
    PyObject* all = PyTuple_New(5);
    if (!all) throw Raised{};
    PyTuple_SET_ITEM(all, 0, THPVariable_Wrap(logprob));
    PyTuple_SET_ITEM(all, 1, THPVariable_Wrap(entropy));
    PyTuple_SET_ITEM(all, 2, THPVariable_Wrap(rank));
    PyTuple_SET_ITEM(all, 3, THPVariable_Wrap(ids));
    PyTuple_SET_ITEM(all, 4, THPVariable_Wrap(values));
    return all;
  });
}

// error class, then the addresses of the entry points in the order of the globals above
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 10;
  if (n != 1 + kEntries) {
    PyErr_SetString(PyExc_TypeError, "bind takes the error class and ten addresses");
    return nullptr;
  }
  void* p[kEntries];
  for (int i = 0; i < kEntries; ++i) {
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
  g_rope = reinterpret_cast<decltype(g_rope)>(p[6]);
  g_rope_rows = reinterpret_cast<decltype(g_rope_rows)>(p[7]);
  g_block_norms = reinterpret_cast<decltype(g_block_norms)>(p[8]);
  g_token_logprobs = reinterpret_cast<decltype(g_token_logprobs)>(p[9]);
  Py_INCREF(a[0]);
  Py_XDECREF(g_error);
  g_error = a[0];
  Py_RETURN_NONE;
}

#define RLDX_METHOD(f) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr }
PyMethodDef g_methods[] = {RLDX_METHOD(bind),          RLDX_METHOD(qkv_rope_append), RLDX_METHOD(kv4_read),
                           RLDX_METHOD(kv4_attention), RLDX_METHOD(sample),          RLDX_METHOD(rope),
                           RLDX_METHOD(rope_rows),     RLDX_METHOD(block_norms),     RLDX_METHOD(token_logprobs),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&g_module); }
