// python_calls.cpp - the host path between Python and the C ABI of include/darkforest_kernels.h.
//
// A decode step or a short sequence keeps the GPU busy for a few microseconds per call, less than an interpreted wrapper
// takes to read a dozen tensors' pointers and to convert the arguments of a ctypes call (7 to 12 us). This module does that
// work - checks, default outputs, the current stream, the call itself with the interpreter lock released - in native code,
// about a microsecond per call before the launch. Behaviour is that of the Python functions in __init__.py, which document
// the arguments and pass them here in order.
//
// The module links no kernel library: bind() receives the addresses of the C functions from the library that the Python
// side loaded, and the exception class that a failed call raises.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>
#include <vector>

#include "../../include/darkforest_kernels.h"

namespace {

// ---------------------------------------------------------------- the bound C functions
#define DF_FUNCTIONS(X)                                                                                                     \
  X(df_attn_forward_block) X(df_attn_forward_bf16) X(df_attn_backward) X(df_attn_backward_bf16) X(df_attn_backward_block)    \
  X(df_attn_backward_block_bf16) X(df_attn_backward_static_scratch) X(df_attn_delta) X(df_attn_delta_bf16) X(df_attn_decode) \
  X(df_attn_merge_partials) X(df_attn_accumulate) X(df_linear_qkv_forward) X(df_linear_forward) X(df_linear_gelu_forward)    \
  X(df_chunked_logit_ce) X(df_layernorm_forward) X(df_layernorm_backward) X(df_gelu_forward) X(df_gelu_backward)             \
  X(df_adamw_update) X(df_adamw_update_multi) X(launch_fused_attention) X(launch_fused_mha_forward)                          \
  X(launch_attention_backward) X(launch_fused_mha_backward) X(df_attn_last_status) X(df_attn_status_string)                  \
  X(df_cache_plan) X(df_cache_release) X(df_cache_append) X(df_cache_attention) X(df_token_logprobs)                        \
  X(df_token_logprobs_backward) X(df_linear_cross_entropy_workspace_bytes) X(df_linear_cross_entropy)                       \
  X(df_linear_cross_entropy_backward) X(df_orthogonalize_workspace_bytes) X(df_orthogonalize) X(df_muon_update)

struct Functions {
#define X(name) decltype(&::name) name = nullptr;
  DF_FUNCTIONS(X)
#undef X
} fn;
PyObject *attention_error = nullptr;  // AttentionError of the package

struct PythonError {};  // a Python exception is set

[[noreturn]] void raise(PyObject *type, const char *text) {
  PyErr_SetString(type, text);
  throw PythonError();
}

// ---------------------------------------------------------------- arguments
const at::Tensor &tensor(PyObject *o) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "expected a torch tensor");
  return THPVariable_Unpack(o);
}

// Device address of a tensor argument; None is a null pointer.
template <typename T = float>
T *ptr(PyObject *o) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = tensor(o);
  if (!t.is_cuda()) raise(attention_error, "attention tensors must live on a CUDA device (no CPU path)");
  if (!t.is_contiguous()) raise(attention_error, "attention tensors must be contiguous");
  return static_cast<T *>(t.data_ptr());
}

uint64_t whole(PyObject *o) {
  if (PyLong_CheckExact(o)) {
    const unsigned long long v = PyLong_AsUnsignedLongLongMask(o);
    if (v == ~0ull && PyErr_Occurred()) throw PythonError();
    return v;
  }
  PyObject *n = PyNumber_Long(o);
  if (!n) throw PythonError();
  const unsigned long long v = PyLong_AsUnsignedLongLongMask(n);
  Py_DECREF(n);
  return v;
}
uint32_t u32(PyObject *o) { return static_cast<uint32_t>(whole(o)); }
float real(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return static_cast<float>(v);
}
uint32_t truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PythonError();
  return static_cast<uint32_t>(v);
}

void *stream(PyObject *o) {
  if (o == Py_None) return static_cast<void *>(c10::cuda::getCurrentCUDAStream().stream());
  PyObject *v = PyObject_GetAttrString(o, "cuda_stream");
  if (!v) throw PythonError();
  const uint64_t s = whole(v);
  Py_DECREF(v);
  return reinterpret_cast<void *>(s);
}

struct Shape3 { uint32_t batch, seq, width; };
Shape3 shape3(PyObject *o) {
  const at::Tensor &t = tensor(o);
  if (t.dim() != 3) raise(PyExc_ValueError, "expected a [batch, seq, heads * d_head] tensor");
  return {static_cast<uint32_t>(t.size(0)), static_cast<uint32_t>(t.size(1)), static_cast<uint32_t>(t.size(2))};
}
struct Shape2 { uint32_t rows, cols; };
Shape2 shape2(PyObject *o) {
  const at::Tensor &t = tensor(o);
  if (t.dim() != 2) raise(PyExc_ValueError, "expected a two-dimensional tensor");
  return {static_cast<uint32_t>(t.size(0)), static_cast<uint32_t>(t.size(1))};
}
uint32_t head_dim(uint64_t width, uint32_t heads) {
  if (heads == 0) raise(PyExc_ZeroDivisionError, "n_heads is zero");
  return static_cast<uint32_t>(width / heads);
}

// ---------------------------------------------------------------- outputs
// Holds the object that a call returns or writes: the caller's, or a new tensor wrapped for Python.
class Out {
 public:
  Out() = default;
  Out(const Out &) = delete;
  Out &operator=(const Out &) = delete;
  ~Out() { Py_XDECREF(o_); }
  void keep(PyObject *o) { Py_INCREF(o); o_ = o; }
  void wrap(at::Tensor t) {
    o_ = THPVariable_Wrap(std::move(t));
    if (!o_) throw PythonError();
  }
  PyObject *get() const { return o_; }
  PyObject *release() { PyObject *o = o_; o_ = nullptr; return o; }

 private:
  PyObject *o_ = nullptr;
};

void given_or_like(Out &out, PyObject *given, PyObject *model) {
  if (given != Py_None) out.keep(given);
  else out.wrap(at::empty_like(tensor(model)));
}
void given_or_empty(Out &out, PyObject *given, PyObject *model, at::IntArrayRef sizes, at::ScalarType type = at::kFloat) {
  if (given != Py_None) out.keep(given);
  else out.wrap(at::empty(sizes, at::TensorOptions().dtype(type).device(tensor(model).device())));
}
void given_or_typed(Out &out, PyObject *given, PyObject *model, at::ScalarType type) {
  given_or_empty(out, given, model, tensor(model).sizes(), type);
}

PyObject *tuple_of(std::initializer_list<Out *> outs) {
  PyObject *t = PyTuple_New(static_cast<Py_ssize_t>(outs.size()));
  if (!t) throw PythonError();
  Py_ssize_t i = 0;
  for (Out *o : outs) PyTuple_SET_ITEM(t, i++, o->release());
  return t;
}

void check(int status) {
  if (status == DF_OK) return;
  const std::string text = std::string("attention call failed: ") + fn.df_attn_status_string(status) + " (" + std::to_string(status) + ")";
  raise(attention_error, text.c_str());
}

// Runs a C function on a stream (its last argument) with the interpreter lock released and checks its status.
template <typename F, typename... A>
void call(F *f, PyObject *stream_arg, A... args) {
  void *s = stream(stream_arg);
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = f(args..., s);
  Py_END_ALLOW_THREADS
  check(status);
}

using Args = PyObject *const *;

// ---------------------------------------------------------------- attention
PyObject *forward(Args a) {  // q k v n_heads scale causal out lse causal_shift stream
  const Shape3 q = shape3(a[0]);
  const uint32_t seq_k = static_cast<uint32_t>(tensor(a[1]).size(1)), heads = u32(a[3]), d = head_dim(q.width, heads);
  Out out, lse;
  given_or_like(out, a[6], a[0]);
  given_or_empty(lse, a[7], a[0], {q.batch, heads, q.seq});
  call(fn.df_attn_forward_block, a[9], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(out.get()), ptr(lse.get()), q.batch, heads, q.seq, seq_k, d, real(a[4]),
       truth(a[5]), static_cast<int64_t>(whole(a[8])));
  return tuple_of({&out, &lse});
}

PyObject *forward_bf16(Args a) {  // q k v n_heads scale causal out lse causal_shift out_fp32 stream
  if (tensor(a[0]).scalar_type() != at::kBFloat16) raise(attention_error, "forward_bf16 needs bfloat16 tensors");
  const Shape3 q = shape3(a[0]);
  const uint32_t seq_k = static_cast<uint32_t>(tensor(a[1]).size(1)), heads = u32(a[3]), d = head_dim(q.width, heads);
  const uint32_t out_fp32 = truth(a[9]);
  const at::ScalarType type = out_fp32 ? at::kFloat : at::kBFloat16;
  Out out, lse;
  given_or_typed(out, a[6], a[0], type);
  if (tensor(out.get()).scalar_type() != type) raise(attention_error, "forward_bf16: out dtype does not match out_fp32");
  given_or_empty(lse, a[7], a[0], {q.batch, heads, q.seq});
  call(fn.df_attn_forward_bf16, a[10], ptr<void>(a[0]), ptr<void>(a[1]), ptr<void>(a[2]), ptr<void>(out.get()), ptr(lse.get()), q.batch, heads, q.seq,
       seq_k, d, real(a[4]), truth(a[5]), static_cast<int64_t>(whole(a[8])), out_fp32);
  return tuple_of({&out, &lse});
}

PyObject *backward(Args a) {  // q k v out d_out lse n_heads scale causal d_q d_k d_v delta_buf stream
  const Shape3 q = shape3(a[0]);
  const uint32_t heads = u32(a[6]), d = head_dim(q.width, heads);
  Out dq, dk, dv, delta;
  given_or_like(dq, a[9], a[0]);
  given_or_like(dk, a[10], a[1]);
  given_or_like(dv, a[11], a[2]);
  given_or_empty(delta, a[12], a[0], {q.batch, heads, q.seq});
  call(fn.df_attn_backward, a[13], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(a[4]), ptr(a[5]), ptr(dq.get()), ptr(dk.get()), ptr(dv.get()),
       ptr(delta.get()), q.batch, heads, q.seq, d, real(a[7]), truth(a[8]));
  return tuple_of({&dq, &dk, &dv});
}

PyObject *backward_bf16(Args a) {  // as backward
  const Shape3 q = shape3(a[0]);
  const uint32_t heads = u32(a[6]), d = head_dim(q.width, heads);
  Out dq, dk, dv, delta;
  given_or_like(dq, a[9], a[0]);
  given_or_like(dk, a[10], a[1]);
  given_or_like(dv, a[11], a[2]);
  given_or_empty(delta, a[12], a[0], {q.batch, heads, q.seq});
  call(fn.df_attn_backward_bf16, a[13], ptr<void>(a[0]), ptr<void>(a[1]), ptr<void>(a[2]), ptr<void>(a[3]), ptr<void>(a[4]), ptr(a[5]),
       ptr<void>(dq.get()), ptr<void>(dk.get()), ptr<void>(dv.get()), ptr(delta.get()), q.batch, heads, q.seq, d, real(a[7]), truth(a[8]));
  return tuple_of({&dq, &dk, &dv});
}

PyObject *backward_static_scratch(Args a) {  // q k v out d_out lse n_heads scale causal d_q d_k d_v stream
  const Shape3 q = shape3(a[0]);
  const uint32_t heads = u32(a[6]), d = head_dim(q.width, heads);
  Out dq, dk, dv;
  given_or_like(dq, a[9], a[0]);
  given_or_like(dk, a[10], a[1]);
  given_or_like(dv, a[11], a[2]);
  call(fn.df_attn_backward_static_scratch, a[12], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(a[4]), ptr(a[5]), ptr(dq.get()), ptr(dk.get()),
       ptr(dv.get()), q.batch, heads, q.seq, d, real(a[7]), truth(a[8]));
  return tuple_of({&dq, &dk, &dv});
}

PyObject *backward_block(Args a) {  // q k v d_out lse delta_buf n_heads scale causal causal_shift d_q d_k d_v stream
  const Shape3 q = shape3(a[0]);
  const uint32_t seq_k = static_cast<uint32_t>(tensor(a[1]).size(1)), heads = u32(a[6]), d = head_dim(q.width, heads);
  Out dq, dk, dv;
  given_or_like(dq, a[10], a[0]);
  given_or_like(dk, a[11], a[1]);
  given_or_like(dv, a[12], a[2]);
  call(fn.df_attn_backward_block, a[13], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(a[4]), ptr(a[5]), ptr(dq.get()), ptr(dk.get()), ptr(dv.get()),
       q.batch, heads, q.seq, seq_k, d, real(a[7]), truth(a[8]), static_cast<int64_t>(whole(a[9])));
  return tuple_of({&dq, &dk, &dv});
}

PyObject *backward_block_bf16(Args a) {  // as backward_block, with out_fp32 before stream
  const Shape3 q = shape3(a[0]);
  const uint32_t seq_k = static_cast<uint32_t>(tensor(a[1]).size(1)), heads = u32(a[6]), d = head_dim(q.width, heads);
  const uint32_t out_fp32 = truth(a[13]);
  const at::ScalarType type = out_fp32 ? at::kFloat : at::kBFloat16;
  Out dq, dk, dv;
  given_or_typed(dq, a[10], a[0], type);
  given_or_typed(dk, a[11], a[1], type);
  given_or_typed(dv, a[12], a[2], type);
  call(fn.df_attn_backward_block_bf16, a[14], ptr<void>(a[0]), ptr<void>(a[1]), ptr<void>(a[2]), ptr<void>(a[3]), ptr(a[4]), ptr(a[5]),
       ptr<void>(dq.get()), ptr<void>(dk.get()), ptr<void>(dv.get()), q.batch, heads, q.seq, seq_k, d, real(a[7]), truth(a[8]),
       static_cast<int64_t>(whole(a[9])), out_fp32);
  return tuple_of({&dq, &dk, &dv});
}

PyObject *delta(Args a) {  // out d_out n_heads delta_buf stream
  const Shape3 o = shape3(a[0]);
  const uint32_t heads = u32(a[2]), d = head_dim(o.width, heads);
  Out buf;
  given_or_empty(buf, a[3], a[0], {o.batch, heads, o.seq});
  call(fn.df_attn_delta, a[4], ptr(a[0]), ptr(a[1]), ptr(buf.get()), o.batch, heads, o.seq, d);
  return buf.release();
}

PyObject *delta_bf16(Args a) {  // as delta
  const Shape3 o = shape3(a[0]);
  const uint32_t heads = u32(a[2]), d = head_dim(o.width, heads);
  Out buf;
  given_or_empty(buf, a[3], a[0], {o.batch, heads, o.seq});
  call(fn.df_attn_delta_bf16, a[4], ptr<void>(a[0]), ptr<void>(a[1]), ptr(buf.get()), o.batch, heads, o.seq, d);
  return buf.release();
}

PyObject *decode(Args a) {  // q k v n_heads cur_seq_len scale block_table page_size partials max_chunks out stream
  const uint32_t heads = u32(a[3]), d = head_dim(static_cast<uint64_t>(tensor(a[0]).numel()), heads);
  Out out;
  given_or_like(out, a[10], a[0]);
  float *part[3] = {nullptr, nullptr, nullptr};
  if (a[8] != Py_None) {
    PyObject *seq = PySequence_Fast(a[8], "partials is a sequence of three tensors");
    if (!seq) throw PythonError();
    const bool three = PySequence_Fast_GET_SIZE(seq) == 3;
    try {
      for (int i = 0; three && i < 3; ++i) part[i] = ptr(PySequence_Fast_GET_ITEM(seq, i));
    } catch (...) {
      Py_DECREF(seq);
      throw;
    }
    Py_DECREF(seq);
    if (!three) raise(PyExc_ValueError, "partials is a sequence of three tensors");
  }
  call(fn.df_attn_decode, a[11], ptr(a[0]), ptr<void>(a[1]), ptr<void>(a[2]), ptr<int32_t>(a[6]), ptr(out.get()), part[0], part[1], part[2], u32(a[9]), heads,
       u32(a[4]), d, real(a[5]), u32(a[7]), tensor(a[1]).scalar_type() == at::kBFloat16 ? 1u : 0u);
  return out.release();
}

PyObject *merge_partials(Args a) {  // o_a lse_a o_b lse_b n_heads stream
  const Shape3 o = shape3(a[0]);
  const uint32_t heads = u32(a[4]), d = head_dim(o.width, heads);
  call(fn.df_attn_merge_partials, a[5], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), o.batch, heads, o.seq, d);
  return PyTuple_Pack(2, a[0], a[1]);
}

PyObject *accumulate(Args a) {  // dst src stream
  call(fn.df_attn_accumulate, a[2], ptr(a[0]), ptr(a[1]), static_cast<uint64_t>(tensor(a[0]).numel()));
  Py_INCREF(a[0]);
  return a[0];
}

// ---------------------------------------------------------------- projections, loss head
PyObject *linear_qkv(Args a) {  // x wq wk wv bq bk bv q k v stream
  const Shape2 x = shape2(a[0]);
  const uint32_t n = static_cast<uint32_t>(tensor(a[1]).size(0));
  Out q, k, v;
  given_or_empty(q, a[7], a[0], {x.rows, n});
  given_or_empty(k, a[8], a[0], {x.rows, n});
  given_or_empty(v, a[9], a[0], {x.rows, n});
  call(fn.df_linear_qkv_forward, a[10], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(a[4]), ptr(a[5]), ptr(a[6]), ptr(q.get()), ptr(k.get()), ptr(v.get()),
       x.rows, x.cols, n);
  return tuple_of({&q, &k, &v});
}

PyObject *linear(Args a) {  // x w bias residual out stream
  const Shape2 x = shape2(a[0]);
  const uint32_t n = static_cast<uint32_t>(tensor(a[1]).size(0));
  Out out;
  given_or_empty(out, a[4], a[0], {x.rows, n});
  call(fn.df_linear_forward, a[5], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(out.get()), x.rows, x.cols, n);
  return out.release();
}

PyObject *linear_gelu(Args a) {  // x w bias pre_activation out keep_pre_activation stream
  const Shape2 x = shape2(a[0]);
  const uint32_t n = static_cast<uint32_t>(tensor(a[1]).size(0));
  Out out, pre;
  given_or_empty(out, a[4], a[0], {x.rows, n});
  if (a[3] == Py_None && !truth(a[5])) pre.keep(Py_None);
  else given_or_empty(pre, a[3], a[0], {x.rows, n});
  call(fn.df_linear_gelu_forward, a[6], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(pre.get()), ptr(out.get()), x.rows, x.cols, n);
  return tuple_of({&pre, &out});
}

PyObject *chunked_logit_ce(Args a) {  // logits targets loss total_rows grad_logits stream
  const Shape2 z = shape2(a[0]);
  call(fn.df_chunked_logit_ce, a[5], ptr(a[0]), ptr<uint32_t>(a[1]), ptr(a[4]), ptr(a[2]), z.rows, z.cols, u32(a[3]));
  Py_INCREF(a[2]);
  return a[2];
}

// ---------------------------------------------------------------- cache in 8 bits, log probabilities
[[noreturn]] void refuse(const char *what, const char *why) {
  raise(attention_error, (std::string(what) + ": " + why).c_str());
}

// A tensor argument of a known type and shape (-1: any size), on the GPU and contiguous.
template <typename T>
T *typed(PyObject *o, at::ScalarType type, std::initializer_list<int64_t> shape, const char *what) {
  T *p = ptr<T>(o);
  const at::Tensor &t = tensor(o);
  if (t.scalar_type() != type) refuse(what, "wrong dtype");
  if (t.dim() != static_cast<int64_t>(shape.size())) refuse(what, "wrong number of dimensions");
  int i = 0;
  for (int64_t n : shape) {
    if (n >= 0 && t.size(i) != n) refuse(what, "wrong size");
    ++i;
  }
  return p;
}
int32_t *ints(PyObject *o, std::initializer_list<int64_t> shape, const char *what) { return typed<int32_t>(o, at::kInt, shape, what); }
float *floats(PyObject *o, std::initializer_list<int64_t> shape, const char *what) { return typed<float>(o, at::kFloat, shape, what); }

uint32_t below_2_31(int64_t n, const char *what) {
  if (n > 0x7fffffffll) refuse(what, "too large");
  return static_cast<uint32_t>(n);
}

// A two-dimensional fp32 or bf16 tensor whose rows may lie apart (their elements together).
struct Rows {
  const void *data;
  uint32_t rows, cols, bf16;
  uint64_t stride;
};
Rows strided_rows(PyObject *o, const char *what) {
  const at::Tensor &t = tensor(o);
  if (!t.is_cuda()) refuse(what, "must live on a CUDA device (no CPU path)");
  if (t.dim() != 2) refuse(what, "expected a two-dimensional tensor");
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) refuse(what, "expected float32 or bfloat16");
  if (t.size(1) > 1 && t.stride(1) != 1) refuse(what, "the elements of a row must lie together");
  if (t.size(0) > 1 && t.stride(0) < t.size(1)) refuse(what, "rows overlap");
  return {t.data_ptr(), below_2_31(t.size(0), what), below_2_31(t.size(1), what), t.scalar_type() == at::kBFloat16 ? 1u : 0u,
          static_cast<uint64_t>(t.size(0) > 1 ? t.stride(0) : t.size(1))};
}

struct Cache {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  uint32_t pages, heads, page_size, d, format;
};
Cache cache(PyObject *k, PyObject *v, PyObject *k_scale, PyObject *v_scale) {
  const at::Tensor &t = tensor(k);
  const at::ScalarType type = t.scalar_type();
  if (type != at::kChar && type != at::kFloat8_e4m3fn) refuse("k_cache", "expected int8 or float8_e4m3fn");
  if (t.dim() != 4) refuse("k_cache", "expected [pages, kv_heads, page_size, d_head]");
  Cache c;
  c.k = typed<uint8_t>(k, type, {-1, -1, -1, -1}, "k_cache");
  c.v = typed<uint8_t>(v, type, {t.size(0), t.size(1), t.size(2), t.size(3)}, "v_cache");
  c.k_scale = floats(k_scale, {t.size(0), t.size(1)}, "k_scale");
  c.v_scale = floats(v_scale, {t.size(0), t.size(1)}, "v_scale");
  c.pages = below_2_31(t.size(0), "k_cache");
  c.heads = below_2_31(t.size(1), "k_cache");
  c.page_size = below_2_31(t.size(2), "k_cache");
  c.d = below_2_31(t.size(3), "k_cache");
  c.format = type == at::kChar ? DF_CACHE_INT8 : DF_CACHE_E4M3;
  return c;
}

void given_or_ints(Out &out, PyObject *given, PyObject *model, std::initializer_list<int64_t> shape, const char *what) {
  given_or_empty(out, given, model, shape, at::kInt);
  ints(out.get(), shape, what);
}
void given_or_floats(Out &out, PyObject *given, PyObject *model, std::initializer_list<int64_t> shape, const char *what) {
  given_or_empty(out, given, model, shape);
  floats(out.get(), shape, what);
}

PyObject *cache_plan(Args a) {  // lens new_tokens block_table free_pages free_count page_size n_tokens lens_out starts slots positions state stream
  int32_t *lens = ints(a[0], {-1}, "lens");
  const int64_t n = tensor(a[0]).size(0), tokens = static_cast<int64_t>(whole(a[6]));
  if (tokens < 0) refuse("n_tokens", "negative");
  int32_t *new_tokens = ints(a[1], {n}, "new_tokens"), *table = ints(a[2], {n, -1}, "block_table");
  int32_t *free_pages = ints(a[3], {-1}, "free_pages"), *free_count = ints(a[4], {1}, "free_count");
  Out lens_out, starts, slots, positions, state;
  given_or_ints(lens_out, a[7], a[0], {n}, "lens_out");
  given_or_ints(starts, a[8], a[0], {n + 1}, "starts");
  given_or_ints(slots, a[9], a[0], {tokens}, "slots");
  given_or_ints(positions, a[10], a[0], {tokens}, "positions");
  given_or_ints(state, a[11], a[0], {2}, "state");
  call(fn.df_cache_plan, a[12], lens, new_tokens, table, free_pages, free_count, ptr<int32_t>(lens_out.get()), ptr<int32_t>(starts.get()),
       ptr<int32_t>(slots.get()), ptr<int32_t>(positions.get()), ptr<int32_t>(state.get()), below_2_31(n, "lens"), below_2_31(tokens, "n_tokens"),
       below_2_31(tensor(a[2]).size(1), "block_table"), u32(a[5]), below_2_31(tensor(a[3]).size(0), "free_pages"));
  return tuple_of({&lens_out, &starts, &slots, &positions, &state});
}

PyObject *cache_release(Args a) {  // lens finished block_table free_pages free_count page_size lens_out count_out stream
  int32_t *lens = ints(a[0], {-1}, "lens");
  const int64_t n = tensor(a[0]).size(0);
  int32_t *finished = ints(a[1], {n}, "finished"), *table = ints(a[2], {n, -1}, "block_table");
  int32_t *free_pages = ints(a[3], {-1}, "free_pages"), *free_count = ints(a[4], {1}, "free_count");
  Out lens_out, count_out;
  given_or_ints(lens_out, a[6], a[0], {n}, "lens_out");
  given_or_ints(count_out, a[7], a[0], {1}, "count_out");
  call(fn.df_cache_release, a[8], lens, finished, table, free_pages, free_count, ptr<int32_t>(lens_out.get()), ptr<int32_t>(count_out.get()),
       below_2_31(n, "lens"), below_2_31(tensor(a[2]).size(1), "block_table"), u32(a[5]), below_2_31(tensor(a[3]).size(0), "free_pages"));
  return tuple_of({&lens_out, &count_out});
}

PyObject *cache_append(Args a) {  // k v slots k_cache v_cache k_scale v_scale stream
  const Rows k = strided_rows(a[0], "k"), v = strided_rows(a[1], "v");
  const Cache c = cache(a[3], a[4], a[5], a[6]);
  if (static_cast<uint64_t>(k.cols) != static_cast<uint64_t>(c.heads) * c.d) refuse("k", "expected kv_heads * d_head columns");
  if (v.rows != k.rows || v.cols != k.cols || v.bf16 != k.bf16) refuse("v", "shape or dtype differs from k");
  int32_t *slots = ints(a[2], {k.rows}, "slots");
  call(fn.df_cache_append, a[7], k.data, v.data, slots, static_cast<void *>(c.k), static_cast<void *>(c.v), c.k_scale, c.v_scale, k.rows, c.heads, c.d,
       c.page_size, c.pages, k.stride, v.stride, k.bf16, c.format);
  return PyTuple_Pack(4, a[3], a[4], a[5], a[6]);
}

PyObject *cache_attention(Args a) {  // q k_cache v_cache k_scale v_scale block_table lens starts n_heads scale workspace out lse stream
  const Rows q = strided_rows(a[0], "q");
  const Cache c = cache(a[1], a[2], a[3], a[4]);
  int32_t *lens = ints(a[6], {-1}, "lens");
  const int64_t n = tensor(a[6]).size(0);
  int32_t *table = ints(a[5], {n, -1}, "block_table"), *starts = ints(a[7], {n + 1}, "starts");
  const uint32_t heads = u32(a[8]);
  if (static_cast<uint64_t>(q.cols) != static_cast<uint64_t>(heads) * c.d) refuse("q", "expected n_heads * d_head columns");
  uint8_t *workspace = ptr<uint8_t>(a[10]);
  Out out, lse;
  const at::ScalarType type = q.bf16 ? at::kBFloat16 : at::kFloat;
  given_or_empty(out, a[11], a[0], {static_cast<int64_t>(q.rows), static_cast<int64_t>(q.cols)}, type);
  void *o = typed<void>(out.get(), type, {q.rows, q.cols}, "out");
  given_or_floats(lse, a[12], a[0], {q.rows, heads}, "lse");
  call(fn.df_cache_attention, a[13], q.data, static_cast<const void *>(c.k), static_cast<const void *>(c.v), c.k_scale, c.v_scale, table, lens, starts, o,
       ptr(lse.get()), static_cast<void *>(workspace), static_cast<uint64_t>(tensor(a[10]).nbytes()), below_2_31(n, "lens"), q.rows, heads, c.heads, c.d,
       c.page_size, c.pages, below_2_31(tensor(a[5]).size(1), "block_table"), q.stride, real(a[9]), q.bf16, c.format);
  return tuple_of({&out, &lse});
}

PyObject *token_logprobs(Args a) {  // logits targets scale top_k logp entropy lse top_ids top_logp stream
  const Rows z = strided_rows(a[0], "logits");
  int32_t *targets = ints(a[1], {z.rows}, "targets");
  const int64_t top = static_cast<int64_t>(whole(a[3]));
  if (top < 0 || top > DF_LOGPROBS_MAX_TOP) refuse("top_k", "out of range");
  Out logp, entropy, lse, ids, best;
  given_or_floats(logp, a[4], a[0], {z.rows}, "logp");
  given_or_floats(entropy, a[5], a[0], {z.rows}, "entropy");
  given_or_floats(lse, a[6], a[0], {z.rows}, "lse");
  given_or_ints(ids, a[7], a[0], {z.rows, top}, "top_ids");
  given_or_floats(best, a[8], a[0], {z.rows, top}, "top_logp");
  call(fn.df_token_logprobs, a[9], z.data, targets, ptr(logp.get()), ptr(entropy.get()), ptr(lse.get()), ptr<int32_t>(ids.get()), ptr(best.get()), z.rows, z.cols,
       z.stride, static_cast<uint32_t>(top), real(a[2]), z.bf16);
  return tuple_of({&logp, &entropy, &lse, &ids, &best});
}

PyObject *token_logprobs_backward(Args a) {  // logits targets lse entropy grad_logp grad_entropy scale d_logits stream
  const Rows z = strided_rows(a[0], "logits");
  int32_t *targets = ints(a[1], {z.rows}, "targets");
  float *lse = floats(a[2], {z.rows}, "lse"), *entropy = floats(a[3], {z.rows}, "entropy");
  float *g = a[4] == Py_None ? nullptr : floats(a[4], {z.rows}, "grad_logp"), *h = a[5] == Py_None ? nullptr : floats(a[5], {z.rows}, "grad_entropy");
  Out d;
  given_or_empty(d, a[7], a[0], {static_cast<int64_t>(z.rows), static_cast<int64_t>(z.cols)}, z.bf16 ? at::kBFloat16 : at::kFloat);
  const Rows to = strided_rows(d.get(), "d_logits");
  if (to.rows != z.rows || to.cols != z.cols || to.bf16 != z.bf16) refuse("d_logits", "shape or dtype differs from the logits");
  call(fn.df_token_logprobs_backward, a[8], z.data, targets, lse, entropy, g, h, const_cast<void *>(to.data), z.rows, z.cols, z.stride, to.stride, real(a[6]),
       z.bf16);
  return d.release();
}

// ---------------------------------------------------------------- loss from hidden states, orthogonalised updates
// For the length of a call: its tensors' device, which becomes the current one, and every other tensor of the call has to be there; and its stream, which becomes the
// current one as well. So what the call allocates belongs to that stream and holds nothing that another one still uses.
class OnDevice {
 public:
  OnDevice(PyObject *first, const char *what, PyObject *stream_arg) : device_(of(first, what)), guard_(device_), caller_(c10::cuda::getCurrentCUDAStream()) {
    if (stream_arg != Py_None) there_.reset_stream(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream(stream_arg)), device_.index()));
  }
  // A result goes to a caller on another stream: when it is dropped there, its memory waits for what that stream does with it.
  PyObject *result(Out &out, PyObject *given) const {
    if (given == Py_None && out.get() != Py_None && caller_ != c10::cuda::getCurrentCUDAStream() && tensor(out.get()).nbytes() > 0)
      c10::cuda::CUDACachingAllocator::recordStream(tensor(out.get()).storage().data_ptr(), caller_);
    return out.get();
  }
  void same(PyObject *o, const char *what) const {
    if (o != Py_None && of(o, what) != device_) refuse(what, "on another device than the others");
  }
  // A workspace: the caller's, or one from the allocator.
  void *workspace(Out &held, PyObject *given, uint64_t bytes, uint64_t *size) const {
    if (given != Py_None) {
      same(given, "workspace");
      if (!tensor(given).is_contiguous()) refuse("workspace", "must be contiguous");
      *size = tensor(given).nbytes();
      return tensor(given).data_ptr();
    }
    held.wrap(at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device_)));
    *size = bytes;
    return tensor(held.get()).data_ptr();
  }

 private:
  static c10::Device of(PyObject *o, const char *what) {
    const at::Tensor &t = tensor(o);
    if (!t.is_cuda()) refuse(what, "must live on a CUDA device (no CPU path)");
    return t.device();
  }
  c10::Device device_;
  c10::cuda::CUDAGuard guard_;
  c10::cuda::CUDAStream caller_;
  c10::cuda::OptionalCUDAStreamGuard there_;
};

struct Head {
  Rows x, w;
  int32_t *targets;
};
Head head(const OnDevice &on, Args a) {  // x weight targets
  on.same(a[1], "weight");
  on.same(a[2], "targets");
  const Rows x = strided_rows(a[0], "x"), w = strided_rows(a[1], "weight");
  if (w.cols != x.cols || w.bf16 != x.bf16) refuse("weight", "width or dtype differs from x");
  return {x, w, ints(a[2], {x.rows}, "targets")};
}

PyObject *linear_cross_entropy(Args a) {  // x weight targets scale loss lse workspace stream
  const OnDevice on(a[0], "x", a[7]);
  const Head h = head(on, a);
  Out loss, lse, ws;
  given_or_floats(loss, a[4], a[0], {h.x.rows}, "loss");
  given_or_floats(lse, a[5], a[0], {h.x.rows}, "lse");
  on.same(on.result(loss, a[4]), "loss");
  on.same(on.result(lse, a[5]), "lse");
  uint64_t size = 0;
  void *work = on.workspace(ws, a[6], fn.df_linear_cross_entropy_workspace_bytes(h.x.rows, h.w.rows, h.x.cols, h.x.bf16, 0), &size);
  call(fn.df_linear_cross_entropy, a[7], h.x.data, h.w.data, h.targets, ptr(loss.get()), ptr(lse.get()), work, size, h.x.rows, h.w.rows, h.x.cols, h.x.stride,
       h.w.stride, real(a[3]), h.x.bf16);
  return tuple_of({&loss, &lse});
}

PyObject *linear_cross_entropy_backward(Args a) {  // x weight targets lse grad_loss scale d_x d_weight want_x want_weight workspace stream
  const OnDevice on(a[0], "x", a[11]);
  const Head h = head(on, a);
  on.same(a[3], "lse");
  on.same(a[4], "grad_loss");
  float *lse = floats(a[3], {h.x.rows}, "lse"), *grad = floats(a[4], {h.x.rows}, "grad_loss");
  const at::ScalarType type = h.x.bf16 ? at::kBFloat16 : at::kFloat;
  Out d[2], ws;
  Rows to[2] = {};
  const Rows *like[2] = {&h.x, &h.w};
  const char *names[2] = {"d_x", "d_weight"};
  for (int i = 0; i < 2; ++i) {
    if (!truth(a[8 + i])) {
      d[i].keep(Py_None);
      continue;
    }
    given_or_empty(d[i], a[6 + i], a[0], {static_cast<int64_t>(like[i]->rows), static_cast<int64_t>(like[i]->cols)}, type);
    on.same(on.result(d[i], a[6 + i]), names[i]);
    to[i] = strided_rows(d[i].get(), names[i]);
    if (to[i].rows != like[i]->rows || to[i].cols != like[i]->cols || to[i].bf16 != h.x.bf16) refuse(names[i], "shape or dtype differs from what it is the gradient of");
  }
  uint64_t size = 0;
  void *work = on.workspace(ws, a[10], fn.df_linear_cross_entropy_workspace_bytes(h.x.rows, h.w.rows, h.x.cols, h.x.bf16, 1), &size);
  call(fn.df_linear_cross_entropy_backward, a[11], h.x.data, h.w.data, h.targets, lse, grad, const_cast<void *>(to[0].data), const_cast<void *>(to[1].data), work,
       size, h.x.rows, h.w.rows, h.x.cols, h.x.stride, h.w.stride, to[0].stride, to[1].stride, real(a[5]), h.x.bf16);
  return tuple_of({&d[0], &d[1]});
}

struct Matrices {
  void *data;
  uint32_t n, rows, cols, bf16;
  uint64_t matrix_stride, row_stride;
};
Matrices matrices(PyObject *o, const char *what) {
  const at::Tensor &t = tensor(o);
  const int64_t d = t.dim();
  if (d != 2 && d != 3) refuse(what, "expected [rows, cols] or [n, rows, cols]");
  if (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) refuse(what, "expected float32 or bfloat16");
  if (t.size(d - 1) > 1 && t.stride(d - 1) != 1) refuse(what, "the elements of a row must lie together");
  const int64_t rows = t.size(d - 2), cols = t.size(d - 1);
  const int64_t row_stride = rows > 1 ? t.stride(d - 2) : cols;
  if (row_stride < cols) refuse(what, "rows overlap");
  return {t.data_ptr(), d == 3 ? below_2_31(t.size(0), what) : 1u, below_2_31(rows, what), below_2_31(cols, what), t.scalar_type() == at::kBFloat16 ? 1u : 0u,
          d == 3 && t.size(0) > 1 ? static_cast<uint64_t>(t.stride(0)) : 0, static_cast<uint64_t>(row_stride)};
}

// A count: a whole number, not what is left of one in 32 bits.
uint32_t count(PyObject *o, const char *what) {
  PyObject *n = PyFloat_Check(o) && PyFloat_AS_DOUBLE(o) == std::floor(PyFloat_AS_DOUBLE(o)) ? PyNumber_Long(o) : PyNumber_Index(o);  // 5.0 is one
  if (!n) throw PythonError();
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(n, &overflow);
  Py_DECREF(n);
  if (overflow != 0 || v < 0 || v > 0x7fffffffll) refuse(what, "out of range");
  return static_cast<uint32_t>(v);
}

struct Polynomial {
  float a, b, c;
};
Polynomial polynomial(PyObject *o) {
  PyObject *s = PySequence_Tuple(o);
  if (!s) throw PythonError();
  float v[3] = {};
  const bool three = PyTuple_GET_SIZE(s) == 3;
  try {
    for (int i = 0; three && i < 3; ++i) v[i] = real(PyTuple_GET_ITEM(s, i));
  } catch (...) {
    Py_DECREF(s);
    throw;
  }
  Py_DECREF(s);
  if (!three) refuse("coefficients", "expected three numbers");
  return {v[0], v[1], v[2]};
}

PyObject *orthogonalize(Args a) {  // update steps coefficients eps out workspace stream
  const OnDevice on(a[0], "update", a[6]);
  const Matrices u = matrices(a[0], "update");
  const Polynomial q = polynomial(a[2]);
  Out out, ws;
  given_or_empty(out, a[4], a[0], tensor(a[0]).sizes(), u.bf16 ? at::kBFloat16 : at::kFloat);
  on.same(on.result(out, a[4]), "out");
  const Matrices o = matrices(out.get(), "out");
  if (!tensor(out.get()).sizes().equals(tensor(a[0]).sizes()) || o.bf16 != u.bf16) refuse("out", "shape or dtype differs from update");
  uint64_t size = 0;
  void *work = on.workspace(ws, a[5], fn.df_orthogonalize_workspace_bytes(u.n, u.rows, u.cols), &size);
  call(fn.df_orthogonalize, a[6], static_cast<const void *>(u.data), o.data, work, size, u.n, u.rows, u.cols, u.matrix_stride, u.row_stride, o.matrix_stride,
       o.row_stride, count(a[1], "steps"), q.a, q.b, q.c, real(a[3]), u.bf16);
  return out.release();
}

class Sequence {  // a list or tuple of tensors
 public:
  explicit Sequence(PyObject *o) : s_(PySequence_Tuple(o)) {
    if (!s_) throw PythonError();
  }
  Sequence(const Sequence &) = delete;
  Sequence &operator=(const Sequence &) = delete;
  ~Sequence() { Py_DECREF(s_); }
  Py_ssize_t size() const { return PyTuple_GET_SIZE(s_); }
  PyObject *operator[](Py_ssize_t i) const { return PyTuple_GET_ITEM(s_, i); }

 private:
  PyObject *s_;
};

PyObject *muon_update(Args a) {  // parameters momenta gradients lr momentum weight_decay nesterov update_scale steps coefficients eps workspace stream
  const Sequence p(a[0]), m(a[1]), g(a[2]);
  if (m.size() != p.size() || g.size() != p.size()) refuse("parameters", "as many parameters, momenta and gradients are expected");
  if (p.size() == 0) Py_RETURN_NONE;
  const OnDevice on(p[0], "parameters", a[12]);
  const at::Tensor &first = tensor(p[0]);
  if (first.dim() != 2) refuse("parameters", "expected matrices");
  const int64_t rows = first.size(0), cols = first.size(1);
  std::vector<df_muon_tensor_t> table;
  for (Py_ssize_t i = 0; i < p.size(); ++i) {
    on.same(p[i], "parameters");
    on.same(m[i], "momenta");
    on.same(g[i], "gradients");
    table.push_back({floats(p[i], {rows, cols}, "parameters"), floats(m[i], {rows, cols}, "momenta"), floats(g[i], {rows, cols}, "gradients")});
  }
  const Polynomial q = polynomial(a[9]);
  const uint32_t n = below_2_31(p.size(), "parameters"), r = below_2_31(rows, "parameters"), c = below_2_31(cols, "parameters");
  Out ws;
  uint64_t size = 0;
  void *work = on.workspace(ws, a[11], fn.df_orthogonalize_workspace_bytes(n, r, c), &size);
  call(fn.df_muon_update, a[12], static_cast<const void *>(table.data()), n, r, c, real(a[3]), real(a[4]), real(a[5]), truth(a[6]), real(a[7]), count(a[8], "steps"), q.a, q.b,
       q.c, real(a[10]), work, size);
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------- LayerNorm, GELU, AdamW
PyObject *layernorm(Args a) {  // x gamma beta out means rstds stream
  const Shape2 x = shape2(a[0]);
  Out out, means, rstds;
  given_or_like(out, a[3], a[0]);
  given_or_empty(means, a[4], a[0], {x.rows});
  given_or_empty(rstds, a[5], a[0], {x.rows});
  call(fn.df_layernorm_forward, a[6], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(out.get()), ptr(means.get()), ptr(rstds.get()), x.rows, x.cols);
  return tuple_of({&out, &means, &rstds});
}

PyObject *layernorm_backward(Args a) {  // grad_out x gamma means rstds grad_x grad_gamma grad_beta stream
  const Shape2 x = shape2(a[1]);
  Out gx;
  given_or_like(gx, a[5], a[1]);
  call(fn.df_layernorm_backward, a[8], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), ptr(a[4]), ptr(gx.get()), ptr(a[6]), ptr(a[7]), x.rows, x.cols);
  return gx.release();
}

PyObject *gelu(Args a) {  // x out stream
  Out out;
  given_or_like(out, a[1], a[0]);
  call(fn.df_gelu_forward, a[2], ptr(a[0]), ptr(out.get()), static_cast<uint64_t>(tensor(a[0]).numel()));
  return out.release();
}

PyObject *gelu_backward(Args a) {  // grad_out x grad_x stream
  Out gx;
  given_or_like(gx, a[2], a[1]);
  call(fn.df_gelu_backward, a[3], ptr(a[0]), ptr(a[1]), ptr(gx.get()), static_cast<uint64_t>(tensor(a[1]).numel()));
  return gx.release();
}

PyObject *adamw_update(Args a) {  // p m v g lr beta1 beta2 eps weight_decay bc1 bc2 stream
  call(fn.df_adamw_update, a[11], ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), static_cast<uint64_t>(tensor(a[0]).numel()), real(a[4]), real(a[5]), real(a[6]),
       real(a[7]), real(a[8]), real(a[9]), real(a[10]));
  Py_RETURN_NONE;
}

PyObject *adamw_step(Args a) {  // table n_tensors total_chunks lr beta1 beta2 eps weight_decay bc1 bc2 stream
  call(fn.df_adamw_update_multi, a[10], ptr<df_adamw_tensor_t>(a[0]), u32(a[1]), whole(a[2]), real(a[3]), real(a[4]), real(a[5]), real(a[6]), real(a[7]),
       real(a[8]), real(a[9]));
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------- AttentionContext (legacy symbols, legacy stream)
void expect_shape(PyObject *o, uint32_t rows, uint64_t cols, const char *what) {
  const at::Tensor &t = tensor(o);
  if (t.dim() == 2 && t.size(0) == static_cast<int64_t>(rows) && t.size(1) == static_cast<int64_t>(cols)) return;
  const std::string text = std::string("attention ") + what + " shape mismatch";
  raise(attention_error, text.c_str());
}

// The legacy symbols run on the legacy default stream: work that the caller queued on another stream has to be finished,
// work on the default stream itself is in order already.
void finish_other_stream() {
  const c10::cuda::CUDAStream s = c10::cuda::getCurrentCUDAStream();
  if (s.stream() == nullptr || s.stream() == cudaStreamLegacy) return;
  Py_BEGIN_ALLOW_THREADS
  s.synchronize();
  Py_END_ALLOW_THREADS
}

PyObject *context_forward(Args a) {  // n_heads seq_len d_head q k v scale causal out
  const uint32_t heads = u32(a[0]), seq = u32(a[1]), d = u32(a[2]);
  expect_shape(a[8], seq, static_cast<uint64_t>(heads) * d, "output");
  float *q = ptr(a[3]), *k = ptr(a[4]), *v = ptr(a[5]), *out = ptr(a[8]);
  const float scale = real(a[6]);
  const uint32_t causal = truth(a[7]);
  finish_other_stream();
  Py_BEGIN_ALLOW_THREADS
  if (heads == 1) fn.launch_fused_attention(q, k, v, out, seq, d, scale, causal);  // lib.rs:2055-2065
  else fn.launch_fused_mha_forward(q, k, v, out, heads, seq, d, scale, causal);
  Py_END_ALLOW_THREADS
  check(fn.df_attn_last_status());
  Py_RETURN_NONE;
}

PyObject *context_backward(Args a) {  // n_heads seq_len d_head q k v d_out scale causal d_q d_k d_v probabilities
  const uint32_t heads = u32(a[0]), seq = u32(a[1]), d = u32(a[2]);
  const char *names[3] = {"d_q", "d_k", "d_v"};
  for (int i = 0; i < 3; ++i) expect_shape(a[9 + i], seq, static_cast<uint64_t>(heads) * d, names[i]);
  float *q = ptr(a[3]), *k = ptr(a[4]), *v = ptr(a[5]), *g = ptr(a[6]), *dq = ptr(a[9]), *dk = ptr(a[10]), *dv = ptr(a[11]), *prob = ptr(a[12]);
  const float scale = real(a[7]);
  const uint32_t causal = truth(a[8]);
  finish_other_stream();
  Py_BEGIN_ALLOW_THREADS
  if (heads == 1) fn.launch_attention_backward(q, k, v, g, dq, dk, dv, prob, seq, d, scale, causal);  // lib.rs:2260-2274
  else fn.launch_fused_mha_backward(q, k, v, g, dq, dk, dv, prob, heads, seq, d, scale, causal);
  Py_END_ALLOW_THREADS
  check(fn.df_attn_last_status());
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------- module
PyObject *bind(PyObject *, PyObject *args) {  // ({name: address}, error class)
  PyObject *table, *error;
  if (!PyArg_ParseTuple(args, "O!O", &PyDict_Type, &table, &error)) return nullptr;
#define X(name)                                                                                       \
  {                                                                                                   \
    PyObject *v = PyDict_GetItemString(table, #name);                                                 \
    void *p = v ? PyLong_AsVoidPtr(v) : nullptr;                                                      \
    if (!p) {                                                                                         \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "no address given for " #name);      \
      return nullptr;                                                                                 \
    }                                                                                                 \
    fn.name = reinterpret_cast<decltype(fn.name)>(p);                                                 \
  }
  DF_FUNCTIONS(X)
#undef X
  Py_INCREF(error);
  Py_XSETREF(attention_error, error);
  Py_RETURN_NONE;
}

template <PyObject *(*F)(Args), int N>
PyObject *entry(PyObject *, Args args, Py_ssize_t n) {
  if (n != N || !attention_error) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments, or bind() was not called");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const PythonError &) {
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(&entry<name, n>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    ENTRY(forward, 10), ENTRY(forward_bf16, 11), ENTRY(backward, 14), ENTRY(backward_bf16, 14), ENTRY(backward_static_scratch, 13),
    ENTRY(backward_block, 14), ENTRY(backward_block_bf16, 15), ENTRY(delta, 5), ENTRY(delta_bf16, 5), ENTRY(decode, 12),
    ENTRY(merge_partials, 6), ENTRY(accumulate, 3), ENTRY(linear_qkv, 11), ENTRY(linear, 6), ENTRY(linear_gelu, 7), ENTRY(chunked_logit_ce, 6),
    ENTRY(layernorm, 7), ENTRY(layernorm_backward, 9), ENTRY(gelu, 3), ENTRY(gelu_backward, 4), ENTRY(adamw_update, 12), ENTRY(adamw_step, 11),
    ENTRY(cache_plan, 13), ENTRY(cache_release, 9), ENTRY(cache_append, 8), ENTRY(cache_attention, 14), ENTRY(token_logprobs, 10),
    ENTRY(token_logprobs_backward, 9), ENTRY(linear_cross_entropy, 8), ENTRY(linear_cross_entropy_backward, 12), ENTRY(orthogonalize, 7),
    ENTRY(muon_update, 13),
    ENTRY(context_forward, 9), ENTRY(context_backward, 13), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "df_python_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_df_python_calls(void) { return PyModule_Create(&module); }
