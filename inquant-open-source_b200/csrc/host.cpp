// Host side of the calls a decode loop makes once per layer and token: the checks, the launch structure and the
// launch in native code.  A Python caller spends 8 to 25 us per call on attribute look-ups, shape and stride objects
// and ctypes fields; these functions read the same numbers off the tensors directly.
//
// Every function serves the ordinary case and returns None (or False), with nothing launched and nothing changed,
// for anything else -- other dtypes, tensor subclasses, unaligned rows, wrong shapes: the Python code behind it then
// makes contiguous copies or raises the errors of the interface.  Nothing is kept between calls.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <algorithm>
#include <cmath>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/inquant_b200.h"

namespace {

int (*g_decode)(const inq_decode_args_t*, inq_stream_t) = nullptr;
int (*g_append)(const inq_append_args_t*, inq_stream_t) = nullptr;
PyTypeObject* g_tensor_type = nullptr;

// A plain strided CUDA tensor of exactly torch.Tensor (no subclass, no wrapper of a transform), or nullptr.
const at::Tensor* plain(PyObject* o) {
  if (Py_TYPE(o) != g_tensor_type) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg()) return nullptr;
  return &t;
}
bool aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// [1, heads, tokens, 128] of 16-bit values whose rows are 16-byte vectors
bool dense_rows(const at::Tensor& t, int64_t heads, const at::Tensor& like) {
  return t.dim() == 4 && t.size(0) == 1 && t.size(1) == heads && t.size(3) == 128 && t.scalar_type() == like.scalar_type() &&
         t.device() == like.device() && t.stride(3) == 1 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 && aligned(t);
}
bool integers(PyObject* const* args, const int* at, int n, long long* out) {
  for (int i = 0; i < n; ++i) {
    out[i] = PyLong_AsLongLong(args[at[i]]);
    if (out[i] == -1 && PyErr_Occurred()) return false;
  }
  return true;
}
PyObject* none() { Py_RETURN_NONE; }
// Exceptions of tensor accessors (a wrapper without storage, ...) never cross into Python: the call is not served.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    if (PyErr_Occurred()) return nullptr;
    Py_RETURN_NONE;
  }
}
// The launch itself does not hold the interpreter: it may wait for room in the launch queue.
template <typename F>
int without_gil(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

// bind(address of inq_decode_attention, address of inq_append_token, torch.Tensor)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "bind takes 3 arguments");
  const int at[] = {0, 1};
  long long v[2];
  if (!integers(args, at, 2, v)) return nullptr;
  g_decode = reinterpret_cast<decltype(g_decode)>(v[0]);
  g_append = reinterpret_cast<decltype(g_append)>(v[1]);
  g_tensor_type = reinterpret_cast<PyTypeObject*>(args[2]);
  Py_INCREF(args[2]);
  Py_RETURN_NONE;
}

// append_token(key, value, tail_key, tail_value, sink_key | None, sink_value | None, tail_count, sink_position, status address)
// -> True when the token was written, a negative return code, or None
PyObject* append_token(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "append_token takes 9 arguments");
  const int at[] = {6, 7, 8};
  long long v[3];
  if (!integers(args, at, 3, v)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *key = plain(args[0]), *value = plain(args[1]), *tk = plain(args[2]), *tv = plain(args[3]);
    if (!key || !value || !tk || !tv || tk->dim() != 4) return none();
    const int64_t heads = tk->size(1), channels = tk->size(3), es = tk->element_size(), row = channels * es;
    if (row % 16 || (tk->stride(1) * es) % 16 || (tk->stride(2) * es) % 16 || tk->stride(3) != 1 || !aligned(*tk)) return none();
    if (tv->sizes() != tk->sizes() || tv->strides() != tk->strides() || !aligned(*tv)) return none();
    for (const at::Tensor* t : {key, value})
      if (t->dim() != 4 || t->size(0) != 1 || t->size(1) != heads || t->size(2) != 1 || t->size(3) != channels || t->scalar_type() != tk->scalar_type() ||
          t->device() != tk->device() || t->stride(3) != 1 || (t->stride(1) * es) % 16 || !aligned(*t))
        return none();
    if (key->stride(1) != value->stride(1)) return none();
    inq_append_args_t a = {};
    a.key = key->data_ptr();
    a.value = value->data_ptr();
    a.src_stride_h = key->stride(1) * es;
    a.tail_key = tk->data_ptr();
    a.tail_value = tv->data_ptr();
    a.tail_stride_h = tk->stride(1) * es;
    a.tail_stride_t = tk->stride(2) * es;
    a.tail_position = (int32_t)v[0];
    a.tail_capacity = (int32_t)tk->size(2);
    a.sink_position = (int32_t)v[1];
    if (v[1] >= 0) {
      const at::Tensor *sk = plain(args[4]), *sv = plain(args[5]);
      if (!sk || !sv || sk->dim() != 4 || sv->sizes() != sk->sizes() || sv->strides() != sk->strides() || v[1] >= sk->size(2)) return none();
      a.sink_key = sk->data_ptr();
      a.sink_value = sv->data_ptr();
      a.sink_stride_h = sk->stride(1) * es;
      a.sink_stride_t = sk->stride(2) * es;
    }
    a.heads = (int32_t)heads;
    a.row_bytes = (int32_t)row;
    a.status = reinterpret_cast<int32_t*>(v[2]);
    const auto stream = c10::cuda::getCurrentCUDAStream(tk->device().index()).stream();
    const int rc = without_gil([&] { return g_append(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
  });
}

bool query_ok(const at::Tensor& q) {
  const auto type = q.scalar_type();
  return (type == at::kHalf || type == at::kBFloat16) && aligned(q);
}
void scratch(inq_decode_args_t& a, const long long* v) {   // workspace, floats, counters, status
  a.partials = reinterpret_cast<float*>(v[0]);
  a.partials_floats = v[1];
  a.counters = reinterpret_cast<int32_t*>(v[2]);
  a.status = reinterpret_cast<int32_t*>(v[3]);
}

// decode(query, sink_key, sink_value, residual_key, residual_value, scale, kv_heads, n_blocks, block_tokens, n_pad, value_kind,
//        value_groups, table, roles, value_roles, workspace, floats, counters, status) -> output, a return code, or None
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 19) return PyErr_Format(PyExc_TypeError, "decode takes 19 arguments");
  const double scale = PyFloat_AsDouble(args[5]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  const int at[] = {6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18};
  long long v[13];
  if (!integers(args, at, 13, v)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* q = plain(args[0]);
    const long long kv_heads = v[0], n_blocks = v[1];
    if (!q || q->dim() != 4 || q->size(0) != 1 || q->size(2) != 1 || q->size(3) != 128 || !query_ok(*q)) return none();
    if (q->stride(3) != 1 || q->stride(1) % 8 || q->size(1) < 1 || q->size(1) % kv_heads) return none();
    inq_decode_seq_t s = {};
    int64_t tokens[2] = {0, 0};
    for (int side = 0; side < 2; ++side) {
      PyObject *ko = args[1 + 2 * side], *vo = args[2 + 2 * side];
      if (ko == Py_None && vo == Py_None) continue;
      const at::Tensor *k = plain(ko), *val = plain(vo);
      if (!k || !val || !dense_rows(*k, kv_heads, *q) || !dense_rows(*val, kv_heads, *q) || k->size(2) != val->size(2)) return none();
      tokens[side] = k->size(2);
      if (!tokens[side]) continue;
      (side ? s.tail_key : s.sink_key) = k->data_ptr();
      (side ? s.tail_value : s.sink_value) = val->data_ptr();
      (side ? s.tail_key_stride_h : s.sink_key_stride_h) = k->stride(1);
      (side ? s.tail_key_stride_t : s.sink_key_stride_t) = k->stride(2);
      (side ? s.tail_value_stride_h : s.sink_value_stride_h) = val->stride(1);
      (side ? s.tail_value_stride_t : s.sink_value_stride_t) = val->stride(2);
    }
    if (n_blocks + tokens[0] + tokens[1] == 0) return none();
    at::Tensor out = at::empty(q->sizes(), q->options().memory_format(at::MemoryFormat::Contiguous));
    s.query = q->data_ptr();
    s.output = out.data_ptr();
    s.query_head_stride = q->stride(1);
    s.table = reinterpret_cast<const int64_t*>(v[6]);
    s.roles = reinterpret_cast<const int8_t*>(v[7]);
    s.value_roles = reinterpret_cast<const int8_t*>(v[8]);
    s.n_blocks = (int32_t)n_blocks;
    s.sink_tokens = (int32_t)tokens[0];
    s.tail_tokens = (int32_t)tokens[1];
    inq_decode_args_t a = {};
    a.n_seq = 1;
    a.seq_host = &s;
    a.kv_heads = (int32_t)kv_heads;
    a.q_per_kv = (int32_t)(q->size(1) / kv_heads);
    a.block_tokens = (int32_t)v[2];
    a.n_pad = (int32_t)v[3];
    a.dtype = q->scalar_type() == at::kHalf ? INQ_F16 : INQ_BF16;
    a.scale = (float)scale;
    a.value_kind = (int32_t)v[4];
    a.value_groups = (int32_t)v[5];
    scratch(a, v + 9);
    const auto stream = c10::cuda::getCurrentCUDAStream(q->device().index()).stream();
    const int rc = without_gil([&] { return g_decode(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
  });
}

// paged_decode(query, cache, blocks, dense, output | None, num_pages, tail_tokens, sink_tokens, heads, block_size, page_bytes,
//              offsets, scale, workspace, floats, counters, status) -> output, a return code, or None
PyObject* paged_decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 17) return PyErr_Format(PyExc_TypeError, "paged_decode takes 17 arguments");
  const double scale = PyFloat_AsDouble(args[12]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  const int at[] = {5, 6, 7, 8, 9, 10, 13, 14, 15, 16};
  long long v[10];
  if (!integers(args, at, 10, v)) return nullptr;
  if (!PyTuple_Check(args[11]) || PyTuple_GET_SIZE(args[11]) != 6) return PyErr_Format(PyExc_TypeError, "six page offsets");
  inq_decode_args_t a = {};
  for (int i = 0; i < 6; ++i) {
    a.page_offsets[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[11], i));
    if (a.page_offsets[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *q = plain(args[0]), *cache = plain(args[1]), *blocks = plain(args[2]), *dense = plain(args[3]);
    const long long pages = v[0], tail = v[1], sink = v[2], heads = v[3], block = v[4];
    if (!q || !cache || !blocks || !dense) return none();
    if (cache->device() != q->device() || blocks->device() != q->device() || dense->device() != q->device()) return none();
    if (q->dim() != 3 || q->size(0) != 1 || q->size(2) != 128 || q->scalar_type() != at::kBFloat16 || !q->is_contiguous() || !aligned(*q)) return none();
    if (q->size(1) % heads || q->size(1) / heads < 1 || q->size(1) / heads > 16) return none();
    if (blocks->scalar_type() != at::kInt || dense->scalar_type() != q->scalar_type() || !dense->is_contiguous()) return none();
    if (!aligned(*dense) || !aligned(*cache)) return none();
    if (dense->dim() != 4 || dense->size(0) != 2 || dense->size(1) != heads || dense->size(2) != block + 4 || dense->size(3) != 128) return none();
    if (pages * block + tail == 0 && !sink) return none();
    at::Tensor out;
    if (args[4] == Py_None) {
      out = at::empty(q->sizes(), q->options());
    } else {
      const at::Tensor* given = plain(args[4]);
      if (!given || !given->is_contiguous() || given->device() != q->device()) return none();
      out = *given;
    }
    inq_decode_seq_t s = {};
    const int64_t stride_h = dense->stride(1), stride_t = dense->stride(2), plane = dense->stride(0) * 2;
    char* const base = static_cast<char*>(dense->data_ptr());
    s.query = q->data_ptr();
    s.output = out.data_ptr();
    s.query_head_stride = 128;
    s.pool = static_cast<const uint8_t*>(cache->data_ptr());
    s.page_table = static_cast<const int32_t*>(blocks->data_ptr());
    s.n_blocks = (int32_t)pages;
    s.pool_pages = (int32_t)cache->size(0);
    s.sink_key = base;
    s.sink_value = base + plane;
    s.tail_key = base + 4 * stride_t * 2;
    s.tail_value = base + 4 * stride_t * 2 + plane;
    s.sink_key_stride_h = s.sink_value_stride_h = s.tail_key_stride_h = s.tail_value_stride_h = stride_h;
    s.sink_key_stride_t = s.sink_value_stride_t = s.tail_key_stride_t = s.tail_value_stride_t = stride_t;
    s.sink_tokens = (int32_t)sink;
    s.tail_tokens = (int32_t)tail;
    // packed tokens covered by the exact sink are masked; so are tail tokens that the sink holds
    s.first_visible = (int32_t)sink;
    s.tail_skip = (int32_t)std::max<long long>(0, sink - pages * block);
    a.n_seq = 1;
    a.seq_host = &s;
    a.kv_heads = (int32_t)heads;
    a.q_per_kv = (int32_t)(q->size(1) / heads);
    a.block_tokens = (int32_t)block;
    a.n_pad = 16;
    a.layout = 1;
    a.dtype = INQ_BF16;
    a.scale = (float)scale;
    a.page_bytes = v[5];
    scratch(a, v + 6);
    const auto stream = c10::cuda::getCurrentCUDAStream(q->device().index()).stream();
    const int rc = without_gil([&] { return g_decode(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    if (args[4] != Py_None) {
      Py_INCREF(args[4]);
      return args[4];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// ---------------------------------------------------------------- uncompressed pages and packed prompts
struct DenseCalls {
  int (*attention)(const inq_prompt_args_t*, inq_stream_t);
  int (*weights)(const inq_prompt_args_t*, inq_stream_t);
  int64_t (*prompt_bytes)(int32_t, int32_t, int32_t, int64_t, int64_t, int32_t, int32_t, int32_t);
  int (*paged)(const inq_paged_attention_args_t*, inq_stream_t);
  int64_t (*paged_bytes)(const inq_paged_attention_args_t*);
  int (*evict)(const inq_evict_args_t*, inq_stream_t);
  int64_t (*evict_bytes)(int32_t, int32_t, int32_t, int64_t);
} g_dense = {};

// bind_dense(addresses of inq_prompt_attention, inq_prompt_weights, inq_prompt_workspace_bytes, inq_paged_attention,
//            inq_paged_attention_workspace_bytes, inq_evict_tokens, inq_evict_workspace_bytes)
PyObject* bind_dense(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "bind_dense takes 7 arguments");
  const int at[] = {0, 1, 2, 3, 4, 5, 6};
  long long v[7];
  if (!integers(args, at, 7, v)) return nullptr;
  g_dense.attention = reinterpret_cast<decltype(g_dense.attention)>(v[0]);
  g_dense.weights = reinterpret_cast<decltype(g_dense.weights)>(v[1]);
  g_dense.prompt_bytes = reinterpret_cast<decltype(g_dense.prompt_bytes)>(v[2]);
  g_dense.paged = reinterpret_cast<decltype(g_dense.paged)>(v[3]);
  g_dense.paged_bytes = reinterpret_cast<decltype(g_dense.paged_bytes)>(v[4]);
  g_dense.evict = reinterpret_cast<decltype(g_dense.evict)>(v[5]);
  g_dense.evict_bytes = reinterpret_cast<decltype(g_dense.evict_bytes)>(v[6]);
  Py_RETURN_NONE;
}

// An argument that may be None: whether it is served, and the tensor (nullptr for None).
bool optional(PyObject* o, const at::Tensor*& t) {
  t = o == Py_None ? nullptr : plain(o);
  return o == Py_None || t != nullptr;
}
// None stands for the default of 1 / sqrt(dim)
bool scale_of(PyObject* o, int64_t dim, float& scale) {
  const double given = o == Py_None ? 1.0 / std::sqrt((double)dim) : PyFloat_AsDouble(o);
  if (given == -1.0 && PyErr_Occurred()) PyErr_Clear();
  scale = (float)given;
  return scale > 0.f;
}
bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool like(const at::Tensor& t, const at::Tensor& other) { return t.scalar_type() == other.scalar_type() && t.device() == other.device(); }
// [a, heads, dim] of 16-bit values whose rows are 16-byte vectors
bool rows3(const at::Tensor& t) { return t.dim() == 3 && t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned(t); }
bool rows4(const at::Tensor& t) {
  return t.dim() == 4 && t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0 && aligned(t);
}
// Whether no two elements share memory, of a tensor of up to three axes that is written (strides are never negative).
bool apart(const at::Tensor& t) {
  int64_t strides[3], sizes[3], end = 1;
  int n = 0;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (t.size(i) <= 1) continue;
    int at = n++;
    for (; at > 0 && strides[at - 1] > t.stride(i); --at) {
      strides[at] = strides[at - 1];
      sizes[at] = sizes[at - 1];
    }
    strides[at] = t.stride(i);
    sizes[at] = t.size(i);
  }
  for (int i = 0; i < n; ++i) {
    if (strides[i] < end) return false;
    end += strides[i] * (sizes[i] - 1);
  }
  return true;
}
bool int32_vector(const at::Tensor& t, int64_t n, const at::Tensor& pages) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.device() == pages.device() && t.is_contiguous();
}
bool on_current_device(const at::Tensor& t) { return t.device().index() == c10::cuda::current_device(); }
PyObject* given_or_new(PyObject* given, at::Tensor& t) {
  if (given == Py_None) return THPVariable_Wrap(t);
  Py_INCREF(given);
  return given;
}
at::Tensor bytes_on(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte).memory_format(at::MemoryFormat::Contiguous)); }
at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor& t, at::ScalarType type) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(t.device()));
}

// Query, key and offsets of a packed prompt into `a`; false for what the Python code has to look at.
bool packed(PyObject* const* args, const at::Tensor*& q, const at::Tensor*& k, PyObject* cu, PyObject* cu_k, PyObject* scale, inq_prompt_args_t& a) {
  q = plain(args[0]);
  k = plain(args[1]);
  const at::Tensor *c = plain(cu), *ck = nullptr;
  if (!q || !k || !c || !optional(cu_k, ck)) return false;
  if (!ck) ck = c;
  if (!rows3(*q) || !rows3(*k) || !half_type(*q) || !like(*k, *q) || !on_current_device(*q)) return false;
  const int64_t dim = q->size(2);
  if ((dim != 64 && dim != 128) || k->size(2) != dim || q->size(0) < 1 || k->size(0) < 1 || k->size(1) < 1 || q->size(1) < 1 || q->size(1) % k->size(1)) return false;
  if (q->stride(0) <= 0 || q->stride(1) <= 0 || k->stride(0) <= 0 || k->stride(1) <= 0) return false;
  if (c->dim() != 1 || c->size(0) < 2 || !int32_vector(*c, c->size(0), *q) || !int32_vector(*ck, c->size(0), *q)) return false;
  if (!scale_of(scale, dim, a.scale)) return false;
  a.q = q->data_ptr();
  a.k = k->data_ptr();
  a.q_stride_t = q->stride(0);
  a.q_stride_h = q->stride(1);
  a.k_stride_t = k->stride(0);
  a.k_stride_h = k->stride(1);
  a.cu_q = static_cast<const int32_t*>(c->data_ptr());
  a.cu_k = static_cast<const int32_t*>(ck->data_ptr());
  a.n_seq = (int32_t)(c->size(0) - 1);
  a.q_rows = q->size(0);
  a.k_rows = k->size(0);
  a.q_heads = (int32_t)q->size(1);
  a.kv_heads = (int32_t)k->size(1);
  a.head_dim = (int32_t)dim;
  a.dtype = q->scalar_type() == at::kHalf ? INQ_F16 : INQ_BF16;
  return true;
}
at::Tensor prompt_scratch(inq_prompt_args_t& a, const at::Tensor& q, bool weights) {
  const int64_t need = g_dense.prompt_bytes(a.q_heads, a.kv_heads, a.head_dim, a.q_rows, a.k_rows, a.n_seq, weights, a.window);
  at::Tensor t;
  if (need) {
    t = bytes_on(q, need);
    a.workspace = t.data_ptr();
    a.workspace_bytes = need;
  }
  return t;
}
bool float_rows(const at::Tensor& t, int64_t rows, int64_t columns, const at::Tensor& q) {
  return t.dim() == 2 && t.size(0) == rows && t.size(1) == columns && t.scalar_type() == at::kFloat && t.device() == q.device() && t.stride(1) == 1;
}

// prompt_attention(query, key, value, cu_seqlens, cu_seqlens_k | None, scale | None, out | None, lse | None, status) -> (out, lse), a return
// code, or None
PyObject* prompt_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "prompt_attention takes 9 arguments");
  const int at[] = {8};
  long long v[1];
  if (!integers(args, at, 1, v)) return nullptr;
  return guarded([&]() -> PyObject* {
    inq_prompt_args_t a = {};
    const at::Tensor *q, *k, *value = plain(args[2]), *out, *lse;
    if (!value || !packed(args, q, k, args[3], args[4], args[5], a) || !optional(args[6], out) || !optional(args[7], lse)) return none();
    if (!rows3(*value) || !like(*value, *q) || value->sizes() != k->sizes() || value->stride(0) <= 0 || value->stride(1) <= 0) return none();
    if (out && (!rows3(*out) || !like(*out, *q) || out->sizes() != q->sizes() || out->stride(0) <= 0 || out->stride(1) <= 0 || !apart(*out))) return none();
    if (lse && (!float_rows(*lse, a.q_heads, a.q_rows, *q) || !apart(*lse))) return none();
    at::Tensor o = out ? *out : fresh(q->sizes(), *q, q->scalar_type()), l = lse ? *lse : fresh({a.q_heads, a.q_rows}, *q, at::kFloat);
    a.v = value->data_ptr();
    a.v_stride_t = value->stride(0);
    a.v_stride_h = value->stride(1);
    a.out = o.data_ptr();
    a.o_stride_t = o.stride(0);
    a.o_stride_h = o.stride(1);
    a.lse = static_cast<float*>(l.data_ptr());
    a.lse_stride = l.stride(0);
    a.status = reinterpret_cast<int32_t*>(v[0]);
    const at::Tensor scratch = prompt_scratch(a, *q, false);
    const auto stream = c10::cuda::getCurrentCUDAStream(q->device().index()).stream();
    const int rc = without_gil([&] { return g_dense.attention(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("NN", given_or_new(args[6], o), given_or_new(args[7], l));
  });
}

// prompt_weights(query, key, lse, cu_seqlens, cu_seqlens_k | None, scale | None, window, out | None, status) -> weights, a return code, or None
PyObject* prompt_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "prompt_weights takes 9 arguments");
  const int at[] = {6, 8};
  long long v[2];
  if (!integers(args, at, 2, v)) return nullptr;
  if (v[0] < 0 || v[0] > 0x7fffffff) return none();
  return guarded([&]() -> PyObject* {
    inq_prompt_args_t a = {};
    const at::Tensor *q, *k, *lse = plain(args[2]), *out;
    if (!lse || !packed(args, q, k, args[3], args[4], args[5], a) || !optional(args[7], out)) return none();
    if (!float_rows(*lse, a.q_heads, a.q_rows, *q) || (out && (!float_rows(*out, a.kv_heads, a.k_rows, *q) || !apart(*out)))) return none();
    at::Tensor w = out ? *out : fresh({a.kv_heads, a.k_rows}, *q, at::kFloat);
    a.lse = static_cast<float*>(lse->data_ptr());
    a.lse_stride = lse->stride(0);
    a.weights = static_cast<float*>(w.data_ptr());
    a.weights_stride = w.stride(0);
    a.window = (int32_t)v[0];
    a.status = reinterpret_cast<int32_t*>(v[1]);
    const at::Tensor scratch = prompt_scratch(a, *q, true);
    const auto stream = c10::cuda::getCurrentCUDAStream(q->device().index()).stream();
    const int rc = without_gil([&] { return g_dense.weights(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    return given_or_new(args[7], w);
  });
}

// Pages, table and lengths: what both calls over pages ask of them.
template <typename Args>
bool paged(const at::Tensor* k, const at::Tensor* value, const at::Tensor* table, const at::Tensor* lengths, Args& a) {
  if (!k || !value || !table || !lengths || !rows4(*k) || !rows4(*value) || !half_type(*k) || !like(*value, *k) || value->sizes() != k->sizes()) return false;
  if (k->numel() == 0 || (k->size(3) != 64 && k->size(3) != 128) || !on_current_device(*k)) return false;
  if (table->dim() != 2 || table->scalar_type() != at::kInt || table->device() != k->device() || table->size(0) < 1 || table->size(1) < 1 || table->stride(1) != 1)
    return false;
  if (!int32_vector(*lengths, table->size(0), *k)) return false;
  if (k->size(2) > 0x3fffffff || table->size(0) > 0x3fffffff || table->size(1) > 0x3fffffff) return false;
  a.k = k->data_ptr();
  a.v = value->data_ptr();
  a.k_stride_p = k->stride(0);
  a.k_stride_h = k->stride(1);
  a.k_stride_t = k->stride(2);
  a.v_stride_p = value->stride(0);
  a.v_stride_h = value->stride(1);
  a.v_stride_t = value->stride(2);
  a.table = static_cast<const int32_t*>(table->data_ptr());
  a.lengths = static_cast<const int32_t*>(lengths->data_ptr());
  a.table_stride = table->stride(0);
  a.pages = k->size(0);
  a.requests = (int32_t)table->size(0);
  a.kv_heads = (int32_t)k->size(1);
  a.head_dim = (int32_t)k->size(3);
  a.page_tokens = (int32_t)k->size(2);
  a.table_columns = (int32_t)table->size(1);
  return true;
}
bool state(const at::Tensor& t, at::ScalarType type, int64_t requests, int64_t heads, int64_t columns, const at::Tensor& pages) {
  return t.dim() == 3 && t.size(0) == requests && t.size(1) == heads && t.size(2) >= columns && t.scalar_type() == type && t.device() == pages.device() &&
         t.stride(2) == 1;
}

// paged_attention(query, key_pages, value_pages, block_table, lengths, scale | None, new_key | None, new_value | None, weights | None,
//                 out_weights | None, out | None, status, counters) -> output or (output, out_weights), a return code, or None
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 13) return PyErr_Format(PyExc_TypeError, "paged_attention takes 13 arguments");
  const int at[] = {11};
  long long v[1];
  if (!integers(args, at, 1, v)) return nullptr;
  return guarded([&]() -> PyObject* {
    inq_paged_attention_args_t a = {};
    const at::Tensor* const counters = plain(args[12]);
    if (!counters || counters->scalar_type() != at::kInt || !counters->is_contiguous()) return none();
    const at::Tensor *q = plain(args[0]), *k = plain(args[1]), *new_k, *new_v, *w, *out_w, *out;
    if (!q || !paged(k, plain(args[2]), plain(args[3]), plain(args[4]), a)) return none();
    if (!optional(args[6], new_k) || !optional(args[7], new_v) || !optional(args[8], w) || !optional(args[9], out_w) || !optional(args[10], out)) return none();
    if (!rows3(*q) || !like(*q, *k) || q->size(0) != a.requests || q->size(2) != a.head_dim || q->size(1) < 1 || q->size(1) % a.kv_heads) return none();
    if (!scale_of(args[5], a.head_dim, a.scale) || !new_k != !new_v) return none();
    for (const at::Tensor* t : {new_k, new_v})
      if (t && (!rows3(*t) || !like(*t, *k) || t->size(0) != a.requests || t->size(1) != a.kv_heads || t->size(2) != a.head_dim)) return none();
    if (out && (!rows3(*out) || !like(*out, *q) || out->sizes() != q->sizes() || !apart(*out))) return none();
    PyObject* const weights_given = args[9] != Py_None ? args[9] : args[8];
    if (!out_w) out_w = w;
    for (const at::Tensor* t : {w, out_w})
      if (t && !state(*t, at::kFloat, a.requests, a.kv_heads, (int64_t)a.table_columns * a.page_tokens, *k)) return none();
    if (out_w && !apart(*out_w)) return none();
    at::Tensor o = out ? *out : fresh(q->sizes(), *q, q->scalar_type());
    a.q = q->data_ptr();
    a.q_stride_b = q->stride(0);
    a.q_stride_h = q->stride(1);
    a.out = o.data_ptr();
    a.o_stride_b = o.stride(0);
    a.o_stride_h = o.stride(1);
    if (new_k) {
      a.new_k = new_k->data_ptr();
      a.new_k_stride_b = new_k->stride(0);
      a.new_k_stride_h = new_k->stride(1);
      a.new_v = new_v->data_ptr();
      a.new_v_stride_b = new_v->stride(0);
      a.new_v_stride_h = new_v->stride(1);
    }
    if (w) {
      a.weights = static_cast<const float*>(w->data_ptr());
      a.w_stride_b = w->stride(0);
      a.w_stride_h = w->stride(1);
    }
    if (out_w) {
      a.out_weights = static_cast<float*>(out_w->data_ptr());
      a.ow_stride_b = out_w->stride(0);
      a.ow_stride_h = out_w->stride(1);
    }
    a.q_heads = (int32_t)q->size(1);
    a.dtype = q->scalar_type() == at::kHalf ? INQ_F16 : INQ_BF16;
    a.status = reinterpret_cast<int32_t*>(v[0]);
    if (counters->device() != q->device() || counters->numel() < (int64_t)a.requests * a.kv_heads * ((a.q_heads / a.kv_heads + 15) / 16)) return none();
    a.counters = static_cast<int32_t*>(counters->data_ptr());
    a.workspace_bytes = g_dense.paged_bytes(&a);
    const at::Tensor scratch = bytes_on(*k, a.workspace_bytes);
    a.workspace = scratch.data_ptr();
    const auto stream = c10::cuda::getCurrentCUDAStream(k->device().index()).stream();
    const int rc = without_gil([&] { return g_dense.paged(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    PyObject* const result = given_or_new(args[10], o);
    if (!out_w) return result;
    Py_INCREF(weights_given);
    return Py_BuildValue("NN", result, weights_given);
  });
}

// evict_tokens(key_pages, value_pages, block_table, lengths, weights, positions, seen, budget, sink, recent, out_weights | None,
//              out_positions | None, out_lengths | None, status) -> (lengths, weights, positions), a return code, or None
PyObject* evict_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 14) return PyErr_Format(PyExc_TypeError, "evict_tokens takes 14 arguments");
  const int at[] = {7, 8, 9, 13};
  long long v[4];
  if (!integers(args, at, 4, v)) return nullptr;
  if (v[0] < 1 || v[0] > 0x3fffffff || v[1] < 0 || v[2] < 0 || v[1] > v[0] || v[2] > v[0] - v[1]) return none();
  return guarded([&]() -> PyObject* {
    inq_evict_args_t a = {};
    const at::Tensor *k = plain(args[0]), *lengths = plain(args[3]), *w = plain(args[4]), *p = plain(args[5]), *seen = plain(args[6]), *out_w, *out_p, *out_n;
    if (!paged(k, plain(args[1]), plain(args[2]), lengths, a) || !w || !p || !seen) return none();
    if (!optional(args[10], out_w) || !optional(args[11], out_p) || !optional(args[12], out_n)) return none();
    const int64_t requests = a.requests, heads = a.kv_heads;
    if (!int32_vector(*seen, requests, *k) || !state(*w, at::kFloat, requests, heads, 1, *k) || !state(*p, at::kInt, requests, heads, w->size(2), *k)) return none();
    if ((out_w && !state(*out_w, at::kFloat, requests, heads, v[0], *k)) || (out_p && !state(*out_p, at::kInt, requests, heads, v[0], *k))) return none();
    if ((out_w && !apart(*out_w)) || (out_p && !apart(*out_p))) return none();
    if (out_n && !int32_vector(*out_n, requests, *k)) return none();
    at::Tensor nw = out_w ? *out_w : fresh({requests, heads, v[0]}, *k, at::kFloat), np = out_p ? *out_p : fresh({requests, heads, v[0]}, *k, at::kInt);
    at::Tensor nn = out_n ? *out_n : fresh({requests}, *k, at::kInt);
    a.seen = static_cast<const int32_t*>(seen->data_ptr());
    a.weights = static_cast<const float*>(w->data_ptr());
    a.positions = static_cast<const int32_t*>(p->data_ptr());
    a.out_weights = static_cast<float*>(nw.data_ptr());
    a.out_positions = static_cast<int32_t*>(np.data_ptr());
    a.out_lengths = static_cast<int32_t*>(nn.data_ptr());
    a.w_stride_b = w->stride(0);
    a.w_stride_h = w->stride(1);
    a.p_stride_b = p->stride(0);
    a.p_stride_h = p->stride(1);
    a.ow_stride_b = nw.stride(0);
    a.ow_stride_h = nw.stride(1);
    a.op_stride_b = np.stride(0);
    a.op_stride_h = np.stride(1);
    a.columns = w->size(2);
    a.budget = (int32_t)v[0];
    a.sink = (int32_t)v[1];
    a.recent = (int32_t)v[2];
    a.status = reinterpret_cast<int32_t*>(v[3]);
    a.workspace_bytes = g_dense.evict_bytes(a.requests, a.kv_heads, a.budget, (int64_t)a.table_columns * a.page_tokens);
    const at::Tensor scratch = bytes_on(*k, a.workspace_bytes);
    a.workspace = scratch.data_ptr();
    const auto stream = c10::cuda::getCurrentCUDAStream(k->device().index()).stream();
    const int rc = without_gil([&] { return g_dense.evict(&a, stream); });
    if (rc != INQ_OK) return PyLong_FromLong(rc);
    return Py_BuildValue("NNN", given_or_new(args[12], nn), given_or_new(args[10], nw), given_or_new(args[11], np));
  });
}

// same_objects(list, list) -> whether both hold the same objects in the same order
PyObject* same_objects(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) return PyErr_Format(PyExc_TypeError, "same_objects takes 2 arguments");
  if (!PyList_Check(args[0]) || !PyList_Check(args[1])) Py_RETURN_FALSE;
  const Py_ssize_t count = PyList_GET_SIZE(args[0]);
  if (count != PyList_GET_SIZE(args[1])) Py_RETURN_FALSE;
  for (Py_ssize_t i = 0; i < count; ++i)
    if (PyList_GET_ITEM(args[0], i) != PyList_GET_ITEM(args[1], i)) Py_RETURN_FALSE;
  Py_RETURN_TRUE;
}

PyMethodDef methods[] = {{"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
                         {"append_token", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append_token)), METH_FASTCALL, nullptr},
                         {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL, nullptr},
                         {"paged_decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_decode)), METH_FASTCALL, nullptr},
                         {"bind_dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind_dense)), METH_FASTCALL, nullptr},
                         {"prompt_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prompt_attention)), METH_FASTCALL, nullptr},
                         {"prompt_weights", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(prompt_weights)), METH_FASTCALL, nullptr},
                         {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_attention)), METH_FASTCALL, nullptr},
                         {"evict_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(evict_tokens)), METH_FASTCALL, nullptr},
                         {"same_objects", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(same_objects)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
  PyObject* const created = PyModule_Create(&module);
  // the PyTorch and the Python this was compiled against, compared before the first use
  if (created && PyModule_AddStringConstant(created, "built_for", INQ_BUILT_FOR) < 0) {
    Py_DECREF(created);
    return nullptr;
  }
  return created;
}
