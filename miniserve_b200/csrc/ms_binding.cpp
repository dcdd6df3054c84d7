// Python entry points of the decode-step operators: append_kv,
// prefix_attention and int8_linear.
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
    const at::Tensor &rope = tensor("rope", o[7]);
    check("rope", rope, at::kFloat, dev, {-1, 2, -1});
    if (!rope.is_contiguous())
      refuse(PyExc_ValueError, "rope must be a contiguous [positions, 2, rotary / 2] table (rope_table)");
    if (rope.size(0) < 1 || rope.size(2) < 1 || 2 * rope.size(2) > dim)
      refuse(PyExc_ValueError, "rope rotates ", 2 * rope.size(2), " entries of heads of ", dim, ", at ", rope.size(0),
             " positions");
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
    check("q", q, type, dev, {T, -1, dim});
    if (o[9] == Py_None) {
      q_out = make(q.sizes(), type, dev);
    } else {
      q_out = tensor("q_out", o[9]);
      check("q_out", q_out, type, dev, q.sizes());
      check_writable("q_out", q_out);
      if (q_out.const_data_ptr() == q.const_data_ptr() && !same_strides(q_out, q))
        refuse(PyExc_ValueError, "q_out in place of q must have q's strides");
    }
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

// bind(address of ms_kv_append, ms_prefix_attention, ms_prefix_attention_workspace, ms_int8_linear, ms_int8_workspace)
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long p[5];
  if (!PyArg_ParseTuple(args, "KKKKK", &p[0], &p[1], &p[2], &p[3], &p[4])) return nullptr;
  entries.prefix_attention = reinterpret_cast<decltype(entries.prefix_attention)>(p[1]);
  entries.prefix_attention_workspace = reinterpret_cast<decltype(entries.prefix_attention_workspace)>(p[2]);
  entries.int8_linear = reinterpret_cast<decltype(entries.int8_linear)>(p[3]);
  entries.int8_workspace = reinterpret_cast<decltype(entries.int8_workspace)>(p[4]);
  entries.kv_append = reinterpret_cast<decltype(entries.kv_append)>(p[0]);
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
