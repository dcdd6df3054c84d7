// Python entry points of the decode-step operators: append_kv,
// prefix_attention, int8_linear, append_kv4, read_kv4 and attention_kv4 of the
// 4-bit cache, and verify_drafts.
//
// A decode step makes dozens of these calls and a small batch's kernels take a
// few microseconds, about what the interpreter needs to look at one tensor's
// type, device, shape and strides a few times over.  So the checks that the
// kernels rely on, the allocations and the call of the C entry point are made
// here, on the tensors themselves: an append of 8 tokens takes 6.5 us of host
// time, 22 us with the same checks in Python.
//
// The C entry points are those of libmssample.so, handed over by address
// (bind); nothing here is a second path to the GPU.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cmath>
#include <cstring>
#include <sstream>
#include <string>

#include "../../include/mssample.h"

namespace {

struct Entries {
  decltype(&ms_kv_append) kv_append;
  decltype(&ms_prefix_attention) prefix_attention;
  decltype(&ms_prefix_attention_workspace) prefix_attention_workspace;
  decltype(&ms_int8_linear) int8_linear;
  decltype(&ms_int8_workspace) int8_workspace;
  decltype(&ms_kv4_append) kv4_append;
  decltype(&ms_kv4_read) kv4_read;
  decltype(&ms_kv4_attention) kv4_attention;
  decltype(&ms_kv4_attention_workspace) kv4_attention_workspace;
  decltype(&ms_verify_drafts) verify_drafts;
  decltype(&ms_verify_workspace) verify_workspace;
} entries = {};

// A refused argument: the Python exception and its message.
struct Refusal {
  PyObject *type;
  std::string text;
};
template <typename... P>
[[noreturn]] void refuse(PyObject *type, const P &...parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw Refusal{type, s.str()};
}

const at::Tensor &tensor(const char *name, PyObject *o) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, name, " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor &cuda_tensor(const char *name, PyObject *o) {
  const at::Tensor &t = tensor(name, o);
  if (!t.is_cuda()) refuse(PyExc_TypeError, name, " must be a CUDA tensor");
  return t;
}

// A tensor of the given type, device and shape (-1: any size), contiguous in
// its last dimension.
void check(const char *name, const at::Tensor &t, at::ScalarType type, at::Device device, at::IntArrayRef shape) {
  if (t.scalar_type() != type) refuse(PyExc_TypeError, name, " has dtype ", t.scalar_type(), ", expected ", type);
  if (t.device() != device) refuse(PyExc_ValueError, name, " is on ", t.device(), ", expected ", device);
  bool same = t.dim() == (int64_t)shape.size();
  for (size_t i = 0; same && i < shape.size(); ++i) same = shape[i] < 0 || t.size(i) == shape[i];
  if (!same) refuse(PyExc_ValueError, name, " has shape ", t.sizes(), ", expected ", shape, " (-1: any)");
  if (t.size(-1) > 1 && t.stride(-1) != 1)
    refuse(PyExc_ValueError, name, " must be contiguous in its last dimension");
}
// No two entries of a tensor that is written share memory by a stride of 0.
void check_writable(const char *name, const at::Tensor &t) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) <= 0)
      refuse(PyExc_ValueError, name, " must not repeat its memory (an expanded tensor)");
}

// Whether two tensors of one shape lie alike: a dimension of one entry is never stepped along.
bool same_strides(const at::Tensor &a, const at::Tensor &b) {
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

int half_code(const char *name, const at::Tensor &t) {
  if (t.scalar_type() == at::kBFloat16) return MS_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return MS_DTYPE_F16;
  refuse(PyExc_TypeError, name, " has dtype ", t.scalar_type(), ", expected bfloat16 or float16");
}
int float_code(const char *name, at::ScalarType type) {
  if (type == at::kFloat) return MS_DTYPE_F32;
  if (type == at::kBFloat16) return MS_DTYPE_BF16;
  if (type == at::kHalf) return MS_DTYPE_F16;
  refuse(PyExc_TypeError, name, " ", type, " is not float32, bfloat16 or float16");
}

void check_cache(const at::Tensor &k, const at::Tensor &v) {
  half_code("cache_k", k);
  check("cache_k", k, k.scalar_type(), k.device(), {-1, -1, -1, -1});
  check("cache_v", v, k.scalar_type(), k.device(), k.sizes());
  if (k.numel() == 0)
    refuse(PyExc_ValueError, "the cache must be a non-empty [pages, page_size, kv_heads, head_dim] tensor");
  check_writable("cache_k", k);
  check_writable("cache_v", v);
}

int64_t integer(const char *name, PyObject *o) {
  const int64_t n = PyLong_AsLongLong(o);
  if (n == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, name, " must be an integer");
  }
  return n;
}

at::Tensor make(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(device));
}

struct CallError {
  int code;
};
// A C entry point with the device current, on its current stream, without the
// interpreter's lock.
template <typename F>
void call(at::Device device, F f) {
  const c10::cuda::CUDAGuard guard(device);
  ms_stream_t stream = reinterpret_cast<ms_stream_t>(c10::cuda::getCurrentCUDAStream(device.index()).stream());
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f(stream);
  Py_END_ALLOW_THREADS;
  if (rc != MS_OK) throw CallError{rc};
}

PyObject *pair(PyObject *a, PyObject *b, PyObject *c = nullptr) {
  PyObject *t = a && b ? PyTuple_New(c ? 3 : 2) : nullptr;
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, a);
  PyTuple_SET_ITEM(t, 1, b);
  if (c) PyTuple_SET_ITEM(t, 2, c);
  return t;
}

const at::Tensor &check_rope(PyObject *o, at::Device dev, int64_t dim) {
  const at::Tensor &rope = tensor("rope", o);
  check("rope", rope, at::kFloat, dev, {-1, 2, -1});
  if (!rope.is_contiguous())
    refuse(PyExc_ValueError, "rope must be a contiguous [positions, 2, rotary / 2] table (rope_table)");
  if (rope.size(0) < 1 || rope.size(2) < 1 || 2 * rope.size(2) > dim)
    refuse(PyExc_ValueError, "rope rotates ", 2 * rope.size(2), " entries of heads of ", dim, ", at ", rope.size(0),
           " positions");
  return rope;
}

// The rotated queries' tensor: q_out as given, or a new one.
at::Tensor check_queries(const at::Tensor &q, PyObject *o, at::ScalarType type, at::Device dev, int64_t T, int64_t dim) {
  check("q", q, type, dev, {T, -1, dim});
  if (o == Py_None) return make(q.sizes(), type, dev);
  const at::Tensor &q_out = tensor("q_out", o);
  check("q_out", q_out, type, dev, q.sizes());
  check_writable("q_out", q_out);
  if (q_out.const_data_ptr() == q.const_data_ptr() && !same_strides(q_out, q))
    refuse(PyExc_ValueError, "q_out in place of q must have q's strides");
  return q_out;
}

// (cache_k, cache_v, k, v, slots, q, positions, rope, interleaved, q_out)
PyObject *append_kv(PyObject *const *o) {
  const at::Tensor &ck = cuda_tensor("cache_k", o[0]), &cv = tensor("cache_v", o[1]);
  check_cache(ck, cv);
  const at::ScalarType type = ck.scalar_type();
  const at::Device dev = ck.device();
  const int64_t heads = ck.size(2), dim = ck.size(3);
  const at::Tensor &k = tensor("k", o[2]), &v = tensor("v", o[3]), &slots = tensor("slots", o[4]);
  check("k", k, type, dev, {-1, heads, dim});
  const int64_t T = k.size(0);
  check("v", v, type, dev, {T, heads, dim});
  check("slots", slots, at::kLong, dev, {T});
  ms_kv_append_args a = {};
  a.dtype = half_code("cache_k", ck);
  a.kv_heads = (int32_t)heads, a.head_dim = (int32_t)dim, a.tokens = T;
  const int interleaved = PyObject_IsTrue(o[8]);
  if (interleaved < 0) return nullptr;
  a.interleaved = interleaved;
  if (o[7] != Py_None) {
    const at::Tensor &rope = check_rope(o[7], dev, dim);
    if (o[6] == Py_None) refuse(PyExc_ValueError, "rope needs positions");
    const at::Tensor &positions = tensor("positions", o[6]);
    check("positions", positions, at::kLong, dev, {T});
    a.rotary = (int32_t)(2 * rope.size(2));
    a.positions = positions.const_data_ptr<int64_t>();
    a.table = rope.const_data_ptr<float>(), a.table_rows = rope.size(0);
  }
  at::Tensor q_out;
  if (o[5] != Py_None) {
    const at::Tensor &q = tensor("q", o[5]);
    q_out = check_queries(q, o[9], type, dev, T, dim);
    a.heads = (int32_t)q.size(1);
    a.q = q.const_data_ptr(), a.q_token = q.stride(0), a.q_head = q.stride(1);
    a.q_out = q_out.data_ptr(), a.q_out_token = q_out.stride(0), a.q_out_head = q_out.stride(1);
  } else if (o[9] != Py_None) {
    refuse(PyExc_ValueError, "q_out needs q");
  }
  a.k = k.const_data_ptr(), a.k_token = k.stride(0), a.k_head = k.stride(1);
  a.v = v.const_data_ptr(), a.v_token = v.stride(0), a.v_head = v.stride(1);
  a.cache_k = ck.data_ptr(), a.ck_page = ck.stride(0), a.ck_token = ck.stride(1), a.ck_head = ck.stride(2);
  a.cache_v = cv.data_ptr(), a.cv_page = cv.stride(0), a.cv_token = cv.stride(1), a.cv_head = cv.stride(2);
  a.pages = ck.size(0), a.page_size = ck.size(1);
  a.slots = slots.const_data_ptr<int64_t>();
  at::Tensor status = make({T}, at::kInt, dev);
  a.status = status.data_ptr<int32_t>();
  call(dev, [&](ms_stream_t s) { return entries.kv_append(&a, s); });
  PyObject *first = q_out.defined() ? (o[9] != Py_None ? Py_NewRef(o[9]) : THPVariable_Wrap(q_out)) : Py_NewRef(Py_None);
  return pair(first, THPVariable_Wrap(status));
}

// (q, cache_k, cache_v, pages, lengths, prefix_pages, prefix_length, scale, out)
PyObject *prefix_attention(PyObject *const *o) {
  const at::Tensor &ck = cuda_tensor("cache_k", o[1]), &cv = tensor("cache_v", o[2]);
  check_cache(ck, cv);
  const at::ScalarType type = ck.scalar_type();
  const at::Device dev = ck.device();
  const int64_t kv_heads = ck.size(2), dim = ck.size(3), page_size = ck.size(1);
  const at::Tensor &q = tensor("q", o[0]), &pages = tensor("pages", o[3]), &lengths = tensor("lengths", o[4]);
  check("q", q, type, dev, {-1, -1, dim});
  const int64_t B = q.size(0), heads = q.size(1);
  if (heads < 1 || heads % kv_heads)
    refuse(PyExc_ValueError, "q has ", heads, " heads, expected a multiple of the cache's ", kv_heads);
  check("pages", pages, at::kInt, dev, {B, -1});
  check("lengths", lengths, at::kInt, dev, {B});
  if (dim % 8 || dim > 128) refuse(PyExc_ValueError, "head_dim ", dim, " is not a multiple of 8 up to 128");
  // a dimension of one entry is never stepped along: its stride may be anything
  auto step = [](const at::Tensor &t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  ms_prefix_attention_args a = {};
  a.cache_k = ck.const_data_ptr(), a.ck_page = step(ck, 0), a.ck_token = step(ck, 1), a.ck_head = step(ck, 2);
  a.cache_v = cv.const_data_ptr(), a.cv_page = step(cv, 0), a.cv_token = step(cv, 1), a.cv_head = step(cv, 2);
  if (((a.ck_page | a.ck_token | a.ck_head | a.cv_page | a.cv_token | a.cv_head) & 7) ||
      ((reinterpret_cast<uintptr_t>(a.cache_k) | reinterpret_cast<uintptr_t>(a.cache_v)) & 15))
    refuse(PyExc_ValueError, "the cache's heads must start 16-byte aligned");
  const int64_t prefix = integer("prefix_length", o[6]);
  int64_t room = 0;
  if (o[5] != Py_None) {
    const at::Tensor &p = tensor("prefix_pages", o[5]);
    check("prefix_pages", p, at::kInt, dev, {-1});
    a.prefix_pages = p.const_data_ptr<int32_t>();
    room = p.size(0) * page_size;
  }
  if (prefix < 0 || prefix > room)
    refuse(PyExc_ValueError, "prefix_length ", prefix, " does not fit prefix_pages (", room, " keys)");
  double scale = 1.0 / std::sqrt((double)dim);
  if (o[7] != Py_None) {
    scale = PyFloat_AsDouble(o[7]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!((float)scale > 0.f) || !std::isfinite((float)scale))
      refuse(PyExc_ValueError, "scale must be positive and finite");
  }
  at::Tensor out;
  if (o[8] == Py_None) {
    out = make({B, heads, dim}, type, dev);
  } else {
    out = tensor("out", o[8]);
    check("out", out, type, dev, q.sizes());
    check_writable("out", out);
  }
  at::Tensor lse = make({B, heads}, at::kFloat, dev), status = make({B}, at::kInt, dev);
  a.dtype = half_code("cache_k", ck);
  a.heads = (int32_t)heads, a.kv_heads = (int32_t)kv_heads, a.head_dim = (int32_t)dim, a.rows = B;
  a.q = q.const_data_ptr(), a.q_row = q.stride(0), a.q_head = q.stride(1);
  a.pages = ck.size(0), a.page_size = page_size;
  a.table = pages.const_data_ptr<int32_t>(), a.table_width = pages.size(1);
  a.table_row = B > 1 ? pages.stride(0) : pages.size(1);
  a.lengths = lengths.const_data_ptr<int32_t>();
  a.prefix_length = prefix, a.scale = (float)scale;
  a.out = out.data_ptr(), a.out_row = out.stride(0), a.out_head = out.stride(1);
  a.lse = lse.data_ptr<float>(), a.status = status.data_ptr<int32_t>();
  at::Tensor workspace;
  {
    const c10::cuda::CUDAGuard guard(dev);
    a.workspace_bytes = entries.prefix_attention_workspace(B, a.heads, a.kv_heads, a.head_dim, prefix);
    workspace = make({a.workspace_bytes}, at::kByte, dev);
  }
  a.workspace = workspace.data_ptr();
  call(dev, [&](ms_stream_t s) { return entries.prefix_attention(&a, s); });
  return pair(o[8] != Py_None ? Py_NewRef(o[8]) : THPVariable_Wrap(out), THPVariable_Wrap(lse),
              THPVariable_Wrap(status));
}

int64_t row_pitch(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
void check_rows(const char *name, const at::Tensor &t) {
  if (t.dim() != 2 || t.size(1) < 1) refuse(PyExc_ValueError, name, " must be a [rows, entries] matrix");
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
    refuse(PyExc_ValueError, name, " must have contiguous rows that do not overlap");
}

// (x, weight, scale, bias, out_dtype, out): the last two or one of them may be None
PyObject *int8_linear(PyObject *const *o) {
  const at::Tensor &x = cuda_tensor("x", o[0]), &w = tensor("weight", o[1]), &scale = tensor("scale", o[2]);
  check_rows("x", x);
  check_rows("weight", w);
  const int code = float_code("x's dtype", x.scalar_type());
  const at::Device dev = w.device();
  const int64_t M = x.size(0), K = w.size(1), N = w.size(0);
  check("weight", w, at::kChar, dev, {-1, -1});
  check("scale", scale, at::kFloat, dev, {N});
  if (N > 1 && w.stride(0) % 16) refuse(PyExc_ValueError, "weight's rows must lie a multiple of 16 bytes apart");
  if (x.size(1) != K || x.device() != dev)
    refuse(PyExc_ValueError, "x must be a [M, ", K, "] tensor on ", dev, ", is ", x.sizes(), " on ", x.device());
  at::ScalarType type = at::kFloat;
  at::Tensor out;
  if (o[5] != Py_None) {
    out = cuda_tensor("out", o[5]);
    type = out.scalar_type();
  }
  if (o[4] != Py_None) {
    if (!THPDtype_Check(o[4])) refuse(PyExc_TypeError, "out_dtype must be a torch.dtype");
    const at::ScalarType want = reinterpret_cast<THPDtype *>(o[4])->scalar_type;
    if (out.defined() && want != type) refuse(PyExc_TypeError, "out has dtype ", type, ", expected ", want);
    type = want;
  }
  const int out_code = float_code("out_dtype", type);
  if (out.defined()) {
    check_rows("out", out);
    check("out", out, type, dev, {M, N});
  } else {
    out = make({M, N}, type, dev);
  }
  const float *bias = nullptr;
  if (o[3] != Py_None) {
    const at::Tensor &b = tensor("bias", o[3]);
    check("bias", b, at::kFloat, dev, {N});
    bias = b.const_data_ptr<float>();
  }
  at::Tensor workspace = make({entries.int8_workspace(M, K)}, at::kByte, dev);
  call(dev, [&](ms_stream_t s) {
    return entries.int8_linear(x.const_data_ptr(), code, row_pitch(x), M, w.const_data_ptr<int8_t>(),
                               (row_pitch(w) + 15) / 16 * 16, scale.const_data_ptr<float>(), N, K, bias,
                               out.data_ptr(), out_code, row_pitch(out), workspace.data_ptr(), s);
  });
  return o[5] != Py_None ? Py_NewRef(o[5]) : THPVariable_Wrap(out);
}

// A KvCache4 as its wrapper hands it over: (k_codes, k_params, v_codes, v_params, head_dim, dtype).
constexpr int kCache4 = 6;
struct Cache4 {
  ms_kv4_cache c = {};
  at::ScalarType type;
  at::Device device;
};
Cache4 cache4(PyObject *const *o) {
  const at::Tensor &kc = cuda_tensor("k_codes", o[0]), &kp = tensor("k_params", o[1]), &vc = tensor("v_codes", o[2]),
                   &vp = tensor("v_params", o[3]);
  Cache4 r{{}, at::kBFloat16, kc.device()};
  if (!THPDtype_Check(o[5])) refuse(PyExc_TypeError, "the cache's dtype must be a torch.dtype");
  r.type = reinterpret_cast<THPDtype *>(o[5])->scalar_type;
  if (r.type != at::kBFloat16 && r.type != at::kHalf)
    refuse(PyExc_TypeError, "the cache's dtype is ", r.type, ", expected bfloat16 or float16");
  const int64_t dim = integer("head_dim", o[4]);
  if (dim < 16 || dim % 16 || dim > 128) refuse(PyExc_ValueError, "head_dim ", dim, " is not a multiple of 16 up to 128");
  const int64_t used = (dim + 31) / 32, stored = used < 2 ? 2 : used, groups = stored == 3 ? 4 : stored;
  check("k_codes", kc, at::kByte, r.device, {-1, -1, -1, stored * 16});
  check("k_params", kp, at::kHalf, r.device, {kc.size(0), kc.size(1), kc.size(2), groups, 2});
  check("v_codes", vc, at::kByte, r.device, kc.sizes());
  check("v_params", vp, at::kHalf, r.device, kp.sizes());
  if (kc.numel() == 0) refuse(PyExc_ValueError, "the cache is empty");
  for (const at::Tensor *t : {&kc, &kp, &vc, &vp}) {
    if (!t->is_contiguous()) refuse(PyExc_ValueError, "the cache's tensors must be contiguous");
    const int64_t align = t == &kp || t == &vp ? groups * 4 : 16;
    if (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & (align - 1))
      refuse(PyExc_ValueError, "the cache's codes must start 16-byte aligned, its parameters ", groups * 4, "-byte aligned");
  }
  r.c.pages = kc.size(0), r.c.kv_heads = (int32_t)kc.size(1), r.c.page_size = kc.size(2), r.c.head_dim = (int32_t)dim;
  r.c.k_codes = static_cast<uint8_t *>(kc.data_ptr()), r.c.k_params = kp.data_ptr();
  r.c.v_codes = static_cast<uint8_t *>(vc.data_ptr()), r.c.v_params = vp.data_ptr();
  return r;
}

// (KvCache4, k, v, slots, q, positions, rope, interleaved, q_out)
PyObject *append_kv4(PyObject *const *o) {
  const Cache4 cache = cache4(o);
  o += kCache4;
  const at::ScalarType type = cache.type;
  const at::Device dev = cache.device;
  const int64_t heads = cache.c.kv_heads, dim = cache.c.head_dim;
  const at::Tensor &k = tensor("k", o[0]), &v = tensor("v", o[1]), &slots = tensor("slots", o[2]);
  check("k", k, type, dev, {-1, heads, dim});
  const int64_t T = k.size(0);
  check("v", v, type, dev, {T, heads, dim});
  check("slots", slots, at::kLong, dev, {T});
  ms_kv4_append_args a = {};
  a.dtype = type == at::kHalf ? MS_DTYPE_F16 : MS_DTYPE_BF16;
  a.tokens = T, a.cache = cache.c;
  const int interleaved = PyObject_IsTrue(o[6]);
  if (interleaved < 0) return nullptr;
  a.interleaved = interleaved;
  if (o[5] != Py_None) {
    const at::Tensor &rope = check_rope(o[5], dev, dim);
    if (o[4] == Py_None) refuse(PyExc_ValueError, "rope needs positions");
    const at::Tensor &positions = tensor("positions", o[4]);
    check("positions", positions, at::kLong, dev, {T});
    a.rotary = (int32_t)(2 * rope.size(2));
    a.positions = positions.const_data_ptr<int64_t>();
    a.table = rope.const_data_ptr<float>(), a.table_rows = rope.size(0);
  }
  at::Tensor q_out;
  if (o[3] != Py_None) {
    const at::Tensor &q = tensor("q", o[3]);
    q_out = check_queries(q, o[7], type, dev, T, dim);
    a.heads = (int32_t)q.size(1);
    a.q = q.const_data_ptr(), a.q_token = q.stride(0), a.q_head = q.stride(1);
    a.q_out = q_out.data_ptr(), a.q_out_token = q_out.stride(0), a.q_out_head = q_out.stride(1);
  } else if (o[7] != Py_None) {
    refuse(PyExc_ValueError, "q_out needs q");
  }
  a.k = k.const_data_ptr(), a.k_token = k.stride(0), a.k_head = k.stride(1);
  a.v = v.const_data_ptr(), a.v_token = v.stride(0), a.v_head = v.stride(1);
  a.slots = slots.const_data_ptr<int64_t>();
  at::Tensor status = make({T}, at::kInt, dev);
  a.status = status.data_ptr<int32_t>();
  call(dev, [&](ms_stream_t s) { return entries.kv4_append(&a, s); });
  PyObject *first = q_out.defined() ? (o[7] != Py_None ? Py_NewRef(o[7]) : THPVariable_Wrap(q_out)) : Py_NewRef(Py_None);
  return pair(first, THPVariable_Wrap(status));
}

// (KvCache4, slots, k_out, v_out)
PyObject *read_kv4(PyObject *const *o) {
  const Cache4 cache = cache4(o);
  o += kCache4;
  const at::Device dev = cache.device;
  const at::Tensor &slots = tensor("slots", o[0]);
  check("slots", slots, at::kLong, dev, {-1});
  const int64_t T = slots.size(0), heads = cache.c.kv_heads, dim = cache.c.head_dim;
  at::Tensor out[2];
  for (int i = 0; i < 2; ++i) {
    const char *name = i ? "v_out" : "k_out";
    if (o[1 + i] == Py_None) {
      out[i] = make({T, heads, dim}, cache.type, dev);
    } else {
      out[i] = tensor(name, o[1 + i]);
      check(name, out[i], cache.type, dev, {T, heads, dim});
      check_writable(name, out[i]);
    }
  }
  if (out[0].numel() > 0 && out[0].const_data_ptr() == out[1].const_data_ptr())
    refuse(PyExc_ValueError, "k_out and v_out are the same memory");
  at::Tensor status = make({T}, at::kInt, dev);
  ms_kv4_read_args a = {};
  a.dtype = cache.type == at::kHalf ? MS_DTYPE_F16 : MS_DTYPE_BF16;
  a.tokens = T, a.cache = cache.c, a.slots = slots.const_data_ptr<int64_t>();
  a.k_out = out[0].data_ptr(), a.k_token = out[0].stride(0), a.k_head = out[0].stride(1);
  a.v_out = out[1].data_ptr(), a.v_token = out[1].stride(0), a.v_head = out[1].stride(1);
  a.status = status.data_ptr<int32_t>();
  call(dev, [&](ms_stream_t s) { return entries.kv4_read(&a, s); });
  return pair(o[1] != Py_None ? Py_NewRef(o[1]) : THPVariable_Wrap(out[0]),
              o[2] != Py_None ? Py_NewRef(o[2]) : THPVariable_Wrap(out[1]), THPVariable_Wrap(status));
}

// (KvCache4, q, pages, lengths, scale, out)
PyObject *attention_kv4(PyObject *const *o) {
  const Cache4 cache = cache4(o);
  o += kCache4;
  const at::Device dev = cache.device;
  const int64_t kv_heads = cache.c.kv_heads, dim = cache.c.head_dim;
  const at::Tensor &q = tensor("q", o[0]), &pages = tensor("pages", o[1]), &lengths = tensor("lengths", o[2]);
  const bool several = q.dim() == 4;
  if (several) check("q", q, cache.type, dev, {-1, -1, -1, dim});
  else check("q", q, cache.type, dev, {-1, -1, dim});
  const int64_t B = q.size(0), T = several ? q.size(1) : 1, heads = q.size(several ? 2 : 1);
  if (heads < 1 || heads % kv_heads)
    refuse(PyExc_ValueError, "q has ", heads, " heads, expected a multiple of the cache's ", kv_heads);
  if (T < 1 || T > 1024) refuse(PyExc_ValueError, "q has ", T, " tokens a row, expected 1 to 1024");
  check("pages", pages, at::kInt, dev, {B, -1});
  if (several) check("lengths", lengths, at::kInt, dev, {B, T});
  else check("lengths", lengths, at::kInt, dev, {B});
  double scale = 1.0 / std::sqrt((double)dim);
  if (o[3] != Py_None) {
    scale = PyFloat_AsDouble(o[3]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!((float)scale > 0.f) || !std::isfinite((float)scale))
      refuse(PyExc_ValueError, "scale must be positive and finite");
  }
  at::Tensor out;
  if (o[4] == Py_None) {
    out = make(q.sizes(), cache.type, dev);
  } else {
    out = tensor("out", o[4]);
    check("out", out, cache.type, dev, q.sizes());
    check_writable("out", out);
  }
  at::Tensor lse = make(q.sizes().slice(0, q.dim() - 1), at::kFloat, dev), status = make({B}, at::kInt, dev);
  ms_kv4_attention_args a = {};
  a.dtype = cache.type == at::kHalf ? MS_DTYPE_F16 : MS_DTYPE_BF16;
  a.tokens = (int32_t)T, a.heads = (int32_t)heads, a.rows = B, a.cache = cache.c;
  a.q = q.const_data_ptr(), a.q_row = q.stride(0), a.q_token = several ? q.stride(1) : 0, a.q_head = q.stride(-2);
  a.table = pages.const_data_ptr<int32_t>(), a.table_width = pages.size(1);
  a.table_row = B > 1 ? pages.stride(0) : pages.size(1);
  a.lengths = lengths.const_data_ptr<int32_t>(), a.length_row = B > 1 ? lengths.stride(0) : T;
  a.scale = (float)scale;
  a.out = out.data_ptr(), a.out_row = out.stride(0), a.out_token = several ? out.stride(1) : 0, a.out_head = out.stride(-2);
  a.lse = lse.data_ptr<float>(), a.status = status.data_ptr<int32_t>();
  at::Tensor workspace;
  {
    const c10::cuda::CUDAGuard guard(dev);
    a.workspace_bytes = entries.kv4_attention_workspace(B, a.tokens, a.heads, a.cache.kv_heads, a.cache.head_dim);
    workspace = make({a.workspace_bytes}, at::kByte, dev);
  }
  a.workspace = workspace.data_ptr();
  call(dev, [&](ms_stream_t s) { return entries.kv4_attention(&a, s); });
  return pair(o[4] != Py_None ? Py_NewRef(o[4]) : THPVariable_Wrap(out), THPVariable_Wrap(lse),
              THPVariable_Wrap(status));
}

// (logits, drafts, uniforms, draft_probs, temperature)
PyObject *verify_drafts(PyObject *const *o) {
  const at::Tensor &logits = cuda_tensor("logits", o[0]), &drafts = tensor("drafts", o[1]), &uniforms = tensor("uniforms", o[2]),
                   &heat = tensor("temperature", o[4]);
  const at::Device dev = logits.device();
  ms_verify_args a = {};
  a.dtype = float_code("logits'", logits.scalar_type());
  check("logits", logits, logits.scalar_type(), dev, {-1, -1, -1});
  const int64_t B = logits.size(0), n = logits.size(1) - 1, V = logits.size(2);
  if (n < 0 || n > 255) refuse(PyExc_ValueError, "logits has ", n + 1, " positions a row, expected 1 to 256");
  if (V < 1) refuse(PyExc_ValueError, "logits has no vocabulary");
  check("drafts", drafts, at::kLong, dev, {B, n});
  check("uniforms", uniforms, at::kDouble, dev, {B, n + 1});
  check("temperature", heat, at::kDouble, dev, {B});
  if (o[3] != Py_None) {
    const at::Tensor &q = tensor("draft_probs", o[3]);
    check("draft_probs", q, at::kFloat, dev, {B, n, V});
    a.draft_probs = q.const_data_ptr<float>(), a.probs_row = q.stride(0), a.probs_pos = q.stride(1);
  }
  a.drafts = (int32_t)n, a.rows = B, a.vocab = V;
  a.logits = logits.const_data_ptr(), a.logits_row = logits.stride(0), a.logits_pos = logits.stride(1);
  a.draft_tokens = drafts.const_data_ptr<int64_t>(), a.draft_row = drafts.stride(0);
  a.uniforms = uniforms.const_data_ptr<double>(), a.uniform_row = uniforms.stride(0);
  a.temperature = heat.const_data_ptr<double>();
  at::Tensor tokens = make({B, n + 1}, at::kLong, dev), probs = make({B, n + 1}, at::kFloat, dev),
             counts = make({B}, at::kInt, dev), status = make({B}, at::kInt, dev);
  a.tokens = tokens.data_ptr<int64_t>(), a.probs = probs.data_ptr<float>();
  a.counts = counts.data_ptr<int32_t>(), a.status = status.data_ptr<int32_t>();
  a.workspace_bytes = entries.verify_workspace(B, a.drafts, V);
  at::Tensor workspace = make({a.workspace_bytes}, at::kByte, dev);
  a.workspace = workspace.data_ptr();
  call(dev, [&](ms_stream_t s) { return entries.verify_drafts(&a, s); });
  PyObject *parts[4] = {THPVariable_Wrap(tokens), THPVariable_Wrap(probs), THPVariable_Wrap(counts), THPVariable_Wrap(status)};
  PyObject *all = PyTuple_New(4);
  for (int i = 0; i < 4; ++i) {
    if (all && parts[i]) PyTuple_SET_ITEM(all, i, parts[i]);
    else return nullptr;
  }
  return all;
}

// Arguments counted, exceptions turned into Python's: (type, text) of a
// refusal, (None, code) of an entry point's return.
template <int kCount, PyObject *(*kRun)(PyObject *const *)>
PyObject *entry(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  if (n != kCount || !entries.kv_append) {
    PyErr_SetString(PyExc_RuntimeError, "binding called before bind, or with a wrong number of arguments");
    return nullptr;
  }
  try {
    return kRun(args);
  } catch (const Refusal &r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const CallError &e) {
    PyObject *type = PyObject_GetAttrString(self, "CallError");
    if (type) {
      PyObject *code = PyLong_FromLong(e.code);
      if (code) PyErr_SetObject(type, code);
      Py_XDECREF(code);
      Py_DECREF(type);
    }
  } catch (const std::bad_alloc &) {
    PyErr_NoMemory();
  } catch (const c10::OutOfMemoryError &e) {
    PyObject *torch = PyImport_ImportModule("torch");
    PyObject *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// bind(addresses of the entry points, in the order of Entries)
PyObject *bind(PyObject *, PyObject *args) {
  constexpr Py_ssize_t kEntries = sizeof(Entries) / sizeof(void *);
  if (PyTuple_GET_SIZE(args) != kEntries) {
    PyErr_Format(PyExc_TypeError, "bind takes %zd addresses", kEntries);
    return nullptr;
  }
  void *p[kEntries];
  for (Py_ssize_t i = 0; i < kEntries; ++i) {
    p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args, i));
    if (!p[i] && PyErr_Occurred()) return nullptr;
  }
  std::memcpy(&entries, p, sizeof(entries));
  Py_RETURN_NONE;
}

template <int kCount, PyObject *(*kRun)(PyObject *const *)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<kCount, kRun>));
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "bind(addresses of the library's entry points)"},
    {"append_kv", fast<10, append_kv>(), METH_FASTCALL, "see miniserve_b200.kvcache.append_kv"},
    {"prefix_attention", fast<9, prefix_attention>(), METH_FASTCALL, "see miniserve_b200.attention.prefix_attention"},
    {"int8_linear", fast<6, int8_linear>(), METH_FASTCALL, "see miniserve_b200.int8.Int8Linear"},
    {"append_kv4", fast<kCache4 + 8, append_kv4>(), METH_FASTCALL, "see miniserve_b200.kvcache4.append_kv4"},
    {"read_kv4", fast<kCache4 + 3, read_kv4>(), METH_FASTCALL, "see miniserve_b200.kvcache4.read_kv4"},
    {"attention_kv4", fast<kCache4 + 5, attention_kv4>(), METH_FASTCALL, "see miniserve_b200.attention4.attention_kv4"},
    {"verify_drafts", fast<5, verify_drafts>(), METH_FASTCALL, "see miniserve_b200.verify.verify_drafts"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "Checked entry points of the decode-step operators.", -1,
                      methods};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
  PyObject *m = PyModule_Create(&module);
  if (!m) return nullptr;
  PyObject *error = PyErr_NewException("miniserve_b200._binding.CallError", PyExc_RuntimeError, nullptr);
  if (!error || PyModule_AddObject(m, "CallError", error) < 0 ||
      PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
