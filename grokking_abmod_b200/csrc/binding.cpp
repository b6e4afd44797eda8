// Python binding of the serving operators: checks torch tensors, takes the
// outputs from torch's allocator, and calls the C interface of
// include/meshb200.h on torch's current stream.
//
// A generated token makes a handful of these calls, each a few microseconds of
// GPU work, so their cost on the host counts.  Checking and packing the same
// arguments in Python took 16 us a call of which 5 are the launch.
//
// Every function returns its outputs, or the library's nonzero status as an
// int, which the Python side turns into its exception; arguments that are not
// what they should be raise ValueError here.

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <utility>

#include "meshb200.h"

namespace {

struct BadArgument : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void require(bool ok, const char* message) {
  if (!ok) throw BadArgument(message);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw BadArgument(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

uint32_t element_type(at::ScalarType t, const char* name) {
  switch (t) {
    case at::kFloat: return MB_F32;
    case at::kBFloat16: return MB_BF16;
    case at::kHalf: return MB_F16;
    default: throw BadArgument(std::string(name) + " must be float32, bfloat16 or float16");
  }
}

uint32_t size32(int64_t v, const char* name) {
  if (v < 0 || v > (int64_t)UINT32_MAX) throw BadArgument(std::string(name) + " must be in 0..2^32-1");
  return (uint32_t)v;
}

// An int argument; None gives `otherwise`.
int64_t integer(PyObject* o, int64_t otherwise) {
  if (o == Py_None) return otherwise;
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw BadArgument("sizes must be integers");
  }
  return v;
}

// Elements of the last dimension are adjacent; an empty tensor may say anything.
bool adjacent(const at::Tensor& t) { return t.numel() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1; }

void on_device(const at::Tensor& t, c10::DeviceIndex device) {
  require(t.is_cuda() && t.get_device() == device, "the operands must be on one CUDA device");
}

// The address of an optional vector: null for None.
template <class T>
T* vector_of(PyObject* o, const char* name, at::ScalarType type, int64_t length, c10::DeviceIndex device) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != length || (length > 1 && t.stride(0) != 1))
    throw BadArgument(std::string(name) + " must be a contiguous " + (type == at::kInt ? "int32" : "float32") +
                      " tensor of " + std::to_string(length));
  on_device(t, device);
  return static_cast<T*>(t.data_ptr());
}

struct Place {
  mb_kv_cache cache;
  mb_cache_rows where;
  c10::DeviceIndex device;
};

// cache.k, cache.v, cache.k_scale, cache.v_scale, table, lengths, offsets
Place place(PyObject* const* a, int64_t rows) {
  const at::Tensor &k = tensor(a[0], "cache.k"), &v = tensor(a[1], "cache.v");
  const at::Tensor &ks = tensor(a[2], "cache.k_scale"), &vs = tensor(a[3], "cache.v_scale");
  const at::Tensor &table = tensor(a[4], "table"), &lengths = tensor(a[5], "lengths");
  require(k.is_cuda(), "the cache must be on a CUDA device");
  require(k.scalar_type() == at::kChar && v.scalar_type() == at::kChar && k.dim() == 4 && v.sizes() == k.sizes() &&
              k.is_contiguous() && v.is_contiguous(),
          "cache.k and cache.v must be contiguous int8 tensors [pages][heads][page_tokens][width]");
  const auto scales = k.sizes().slice(0, 2);
  require(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.sizes() == scales &&
              vs.sizes() == scales && ks.is_contiguous() && vs.is_contiguous(),
          "cache.k_scale and cache.v_scale must be contiguous float32 tensors [pages][heads]");
  require(table.scalar_type() == at::kInt && table.dim() == 2 && adjacent(table) && table.stride(0) >= 0,
          "table must be an int32 tensor [batch][pages] with adjacent page numbers");
  Place p;
  p.device = k.get_device();
  for (const at::Tensor* t : {&v, &ks, &vs, &table, &lengths}) on_device(*t, p.device);
  const int64_t batch = table.size(0), pages = table.size(1);
  require(lengths.scalar_type() == at::kInt && lengths.dim() == 1 && lengths.size(0) == batch &&
              (batch <= 1 || lengths.stride(0) == 1),
          "lengths must be a contiguous int32 tensor [batch]");
  p.cache = mb_kv_cache{static_cast<int8_t*>(k.data_ptr()),
                        static_cast<int8_t*>(v.data_ptr()),
                        static_cast<float*>(ks.data_ptr()),
                        static_cast<float*>(vs.data_ptr()),
                        size32(k.size(0), "pages"),
                        size32(k.size(1), "heads"),
                        size32(k.size(2), "page_tokens"),
                        size32(k.size(3), "width")};
  p.where = mb_cache_rows{static_cast<const int32_t*>(table.data_ptr()),
                          static_cast<const int32_t*>(lengths.data_ptr()),
                          vector_of<const int32_t>(a[6], "offsets", at::kInt, batch + 1, p.device),
                          (size_t)(batch > 1 ? table.stride(0) : pages),
                          (size_t)rows,
                          size32(pages, "table pages"),
                          size32(batch, "batch")};
  return p;
}

struct RowView {
  const void* at;
  size_t row, head;
};

RowView rows_of(const at::Tensor& t, const char* name, c10::DeviceIndex device) {
  if (t.dim() != 3 || !adjacent(t) || t.stride(0) < 0 || t.stride(1) < 0)
    throw BadArgument(std::string(name) + " must be [rows][heads][head_dim] with adjacent channels");
  on_device(t, device);
  return RowView{t.data_ptr(), (size_t)t.stride(0), (size_t)t.stride(1)};
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::DeviceIndex device) {
  return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, device), std::nullopt);
}

void* stream_of(c10::DeviceIndex device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

PyObject* tuple_of(std::initializer_list<at::Tensor> items) {
  PyObject* r = PyTuple_New((Py_ssize_t)items.size());
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : items) {
    PyObject* o = THPVariable_Wrap(t);
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// Runs a function's body, turning C++ exceptions into Python's.
template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  if (given != wanted) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const BadArgument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (cache x 4, table, lengths, offsets, k, v, max_new, status)
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const at::Tensor &k = tensor(a[7], "k"), &v = tensor(a[8], "v");
    require(k.dim() == 3 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
            "k and v must be [rows][heads][head_dim] of one shape and type");
    const int64_t rows = k.size(0);
    const Place p = place(a, rows);
    require(k.size(1) == (int64_t)p.cache.heads, "k and v must have the cache's heads");
    const RowView kr = rows_of(k, "k", p.device), vr = rows_of(v, "v", p.device);
    const mb_cache_write_args args{p.cache,
                                   p.where,
                                   kr.at,
                                   vr.at,
                                   kr.row,
                                   kr.head,
                                   vr.row,
                                   vr.head,
                                   vector_of<int>(a[10], "status", at::kInt, 1, p.device),
                                   size32(k.size(2), "head_dim"),
                                   element_type(k.scalar_type(), "k"),
                                   size32(integer(a[9], p.where.offsets ? rows : 1), "max_new"),
                                   0};
    const c10::cuda::CUDAGuard guard(p.device);
    return PyLong_FromLong(mb_op_cache_write(&args, stream_of(p.device)));
  });
}

// (cache x 4, table, lengths, tokens, first, head_dim, dtype, status)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    PyObject* at[7] = {a[0], a[1], a[2], a[3], a[4], a[5], Py_None};
    const Place p = place(at, 0);
    const uint32_t tokens = size32(integer(a[6], 0), "tokens");
    const int64_t batch = p.where.batch, head_dim = integer(a[8], p.cache.width);
    require(head_dim >= 1 && head_dim <= (int64_t)p.cache.width, "head_dim must be in 1..the cache's width");
    at::ScalarType type = at::kFloat;
    if (a[9] != Py_None) {
      if (!THPDtype_Check(a[9])) throw BadArgument("dtype must be a torch dtype");
      type = reinterpret_cast<THPDtype*>(a[9])->scalar_type;
    }
    const uint32_t code = element_type(type, "dtype");
    const c10::cuda::CUDAGuard guard(p.device);
    const int64_t shape[4] = {batch, (int64_t)tokens, (int64_t)p.cache.heads, head_dim};
    at::Tensor k = empty(shape, type, p.device), v = empty(shape, type, p.device);
    const mb_cache_read_args args{p.cache,
                                  p.where,
                                  vector_of<const int32_t>(a[7], "first", at::kInt, batch, p.device),
                                  k.data_ptr(),
                                  v.data_ptr(),
                                  vector_of<int>(a[10], "status", at::kInt, 1, p.device),
                                  (uint32_t)head_dim,
                                  code,
                                  tokens,
                                  0};
    const int status = mb_op_cache_read(&args, stream_of(p.device));
    return status ? PyLong_FromLong(status) : tuple_of({std::move(k), std::move(v)});
  });
}

// (cache x 4, table, lengths, offsets, q, first, scale, max_new, max_tokens, status)
PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor& q = tensor(a[7], "q");
    require(q.dim() == 3, "q must be [rows][q_heads][head_dim]");
    const int64_t rows = q.size(0), heads = q.size(1), head_dim = q.size(2);
    const Place p = place(a, rows);
    const RowView r = rows_of(q, "q", p.device);
    mb_cache_attention_args args{};
    args.cache = p.cache;
    args.where = p.where;
    args.first = vector_of<const int32_t>(a[8], "first", at::kInt, p.where.batch, p.device);
    args.d_status = vector_of<int>(a[12], "status", at::kInt, 1, p.device);
    args.q = r.at;
    args.q_row_stride = r.row;
    args.q_head_stride = r.head;
    args.q_heads = size32(heads, "q_heads");
    args.head_dim = size32(head_dim, "head_dim");
    args.dtype = element_type(q.scalar_type(), "q");
    if (a[9] == Py_None) {
      args.scale = (float)(1.0 / std::sqrt((double)head_dim));
    } else {
      const double scale = PyFloat_AsDouble(a[9]);
      if (scale == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw BadArgument("scale must be a number");
      }
      args.scale = (float)scale;
    }
    args.max_new = size32(integer(a[10], p.where.offsets ? rows : 1), "max_new");
    const int64_t room = (int64_t)p.where.table_pages * p.cache.page_tokens;
    args.max_tokens = size32(integer(a[11], room < INT_MAX ? room : INT_MAX), "max_tokens");
    const c10::cuda::CUDAGuard guard(p.device);
    int status = mb_op_cache_attention_workspace(p.where.batch, (size_t)rows, args.q_heads, p.cache.heads,
                                                 args.head_dim, args.dtype, args.max_new, args.max_tokens,
                                                 &args.workspace_bytes);
    if (status) return PyLong_FromLong(status);
    at::Tensor out = empty(q.sizes(), q.scalar_type(), p.device);
    const int64_t lse_shape[2] = {heads, rows};
    at::Tensor lse = empty(lse_shape, at::kFloat, p.device), work;
    if (args.workspace_bytes) {
      const int64_t bytes = (int64_t)args.workspace_bytes;
      work = empty(bytes, at::kByte, p.device);
      args.workspace = work.data_ptr();
    }
    args.out = out.data_ptr();
    args.lse = static_cast<float*>(lse.data_ptr());
    status = mb_op_cache_attention(&args, stream_of(p.device));
    return status ? PyLong_FromLong(status) : tuple_of({std::move(out), std::move(lse)});
  });
}

struct Logits {
  const at::Tensor* t;
  int64_t rows, vocab;
  size_t stride;
  uint32_t type;
  c10::DeviceIndex device;
};

Logits logits_of(PyObject* o) {
  const at::Tensor& t = tensor(o, "logits");
  require(t.is_cuda() && t.dim() == 2 && adjacent(t) && t.stride(0) >= 0,
          "logits must be a CUDA tensor [rows][vocab] with adjacent columns");
  const int64_t rows = t.size(0), vocab = t.size(1);
  return Logits{&t, rows, vocab, (size_t)(rows > 1 ? t.stride(0) : vocab), element_type(t.scalar_type(), "logits"),
                (c10::DeviceIndex)t.get_device()};
}

// (logits, tokens, top, status)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const Logits x = logits_of(a[0]);
    const uint32_t top = size32(integer(a[2], 0), "top");
    require(top <= 4096, "top must be in 0..32");
    require(a[1] != Py_None, "tokens must be a tensor");
    mb_token_logprobs_args args{};
    args.tokens = vector_of<const int32_t>(a[1], "tokens", at::kInt, x.rows, x.device);
    args.d_status = vector_of<int>(a[3], "status", at::kInt, 1, x.device);
    const c10::cuda::CUDAGuard guard(x.device);
    const int64_t best_shape[2] = {x.rows, (int64_t)top};
    at::Tensor logprob = empty(x.rows, at::kFloat, x.device), entropy = empty(x.rows, at::kFloat, x.device);
    at::Tensor lse = empty(x.rows, at::kFloat, x.device), best = empty(best_shape, at::kFloat, x.device);
    at::Tensor index = empty(best_shape, at::kInt, x.device);
    if (x.rows) {
      args.logits = x.t->data_ptr();
      args.logprob = static_cast<float*>(logprob.data_ptr());
      args.entropy = static_cast<float*>(entropy.data_ptr());
      args.lse = static_cast<float*>(lse.data_ptr());
      args.top_logprob = static_cast<float*>(best.data_ptr());
      args.top_index = static_cast<int32_t*>(index.data_ptr());
      args.row_stride = x.stride;
      args.rows = (size_t)x.rows;
      args.vocab = size32(x.vocab, "vocab");
      args.dtype = x.type;
      args.top = top;
      if (const int status = mb_op_token_logprobs(&args, stream_of(x.device))) return PyLong_FromLong(status);
    }
    return tuple_of({std::move(logprob), std::move(entropy), std::move(lse), std::move(best), std::move(index)});
  });
}

// (logits, tokens, lse, entropy, dlogprob, dentropy, status)
PyObject* token_logprobs_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Logits x = logits_of(a[0]);
    require(a[1] != Py_None && a[2] != Py_None, "tokens and lse must be tensors");
    mb_token_logprobs_backward_args args{};
    args.tokens = vector_of<const int32_t>(a[1], "tokens", at::kInt, x.rows, x.device);
    args.lse = vector_of<const float>(a[2], "lse", at::kFloat, x.rows, x.device);
    args.entropy = vector_of<const float>(a[3], "entropy", at::kFloat, x.rows, x.device);
    args.dlogprob = vector_of<const float>(a[4], "dlogprob", at::kFloat, x.rows, x.device);
    args.dentropy = vector_of<const float>(a[5], "dentropy", at::kFloat, x.rows, x.device);
    args.d_status = vector_of<int>(a[6], "status", at::kInt, 1, x.device);
    const c10::cuda::CUDAGuard guard(x.device);
    const int64_t shape[2] = {x.rows, x.vocab};
    at::Tensor d = empty(shape, x.t->scalar_type(), x.device);
    if (x.rows) {
      args.logits = x.t->data_ptr();
      args.dlogits = d.data_ptr();
      args.row_stride = x.stride;
      args.rows = (size_t)x.rows;
      args.vocab = size32(x.vocab, "vocab");
      args.dtype = x.type;
      if (const int status = mb_op_token_logprobs_backward(&args, stream_of(x.device)))
        return PyLong_FromLong(status);
    }
    return THPVariable_Wrap(std::move(d));
  });
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(cache_write),    METHOD(cache_read),
                         METHOD(cache_attention), METHOD(token_logprobs),
                         METHOD(token_logprobs_backward), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() {
  uint64_t key = 0;
  if (mb_header_key(&key) != 0 || key != MB_HEADER_KEY) {
    PyErr_SetString(PyExc_ImportError,
                    "the library was built from another header (meshb200.h) than its Python binding: build both "
                    "(python -m grokking_abmod_b200.build)");
    return nullptr;
  }
  return PyModule_Create(&module);
}
