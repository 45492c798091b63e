// Host side of the paged cache and of prompt attention: argument checks,
// output allocation and the call into libinnerq_b200.so, as a CPython module
// over torch's C++ tensors.  A decode step makes a handful of these calls per
// layer, and on small batches their host time is what counts: a call takes
// about half of what the same checks cost in Python.
//
// Every function raises TypeError / ValueError / NotImplementedError for bad
// arguments before any launch, and innerq_b200._lib.InnerqError for a status
// of the C ABI.  Inputs whose rows are not contiguous and 16-byte aligned are
// copied first; an output of prompt attention with such rows is written through
// a copy.  Work goes to the current stream of the tensors' device.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/innerq_b200.h"

namespace {

using at::Tensor;

constexpr int64_t kD = 128, kTile = 32, kBlock = 4608;

struct Raise {
  PyObject* type;
  std::string text;
};

// a Python error that is set already
struct Pending {};

// entry points of the library, resolved by bind()
decltype(&innerq_paged_append) f_append = nullptr;
decltype(&innerq_paged_read) f_read = nullptr;
decltype(&innerq_paged_attn_workspace) f_workspace = nullptr;
decltype(&innerq_paged_attn) f_attn = nullptr;
decltype(&innerq_prompt_attn) f_prompt = nullptr;
decltype(&innerq_last_error) f_error = nullptr;

// a failing status of the C ABI as _lib.InnerqError(function, code, message)
struct Failed {
  const char* fn;
  int code;
};

void check(int rc, const char* fn) {
  if (rc != INNERQ_OK) throw Failed{fn, rc};
}

std::string shape(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string type_name(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kFloat: return "float32";
    case at::kInt: return "int32";
    default: return c10::toString(t);
  }
}
std::string kind(const Tensor& t) { return type_name(t.scalar_type()) + " on " + t.device().str(); }

int dtype_code(at::ScalarType t) {
  if (t == at::kHalf) return INNERQ_DT_F16;
  if (t == at::kBFloat16) return INNERQ_DT_BF16;
  throw Raise{PyExc_TypeError, "innerq_b200 kernels take float16 or bfloat16 tensors, got " + type_name(t)};
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Raise{PyExc_TypeError, std::string(what) + " must be a tensor"};
  return THPVariable_Unpack(o);
}
void need_cuda(const Tensor& t, const char* what) {
  if (!t.is_cuda())
    throw Raise{PyExc_RuntimeError, std::string(what) + " must be a CUDA tensor: innerq_b200 has no CPU path"};
}
int64_t integer(PyObject* o, const char* what) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Raise{PyExc_TypeError, std::string(what) + " must be an integer"};
  }
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Pending{};
  return v == 1;
}

float scale_of(PyObject* o) {
  if (o == Py_None) return 1.f / std::sqrt((float)kD);
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Raise{PyExc_TypeError, "scale must be a number"};
  }
  return (float)v;
}

// t as [tokens, heads, 128] with contiguous, 16-byte aligned rows
Tensor rows(const Tensor& t, const char* what, at::ScalarType dtype, at::Device device) {
  if (t.dim() != 3)
    throw Raise{PyExc_ValueError, std::string(what) + " must be [tokens, heads, head_dim], got " + shape(t)};
  if (t.scalar_type() != dtype || t.device() != device)
    throw Raise{PyExc_TypeError, std::string(what) + " is " + kind(t) + ", expected " + type_name(dtype) + " on " + device.str()};
  // a broadcast dimension (stride 0) has no tensor map
  const bool flat = (t.stride(0) == 0 && t.size(0) > 1) || (t.stride(1) == 0 && t.size(1) > 1);
  if (t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && (uintptr_t)t.data_ptr() % 16 == 0 && !flat) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// an int32 vector of n elements (n < 0: any)
Tensor index(const Tensor& t, const char* what, int64_t n, at::Device device) {
  if (t.dim() != 1 || (n >= 0 && t.size(0) != n))
    throw Raise{PyExc_ValueError, std::string(what) + " must have " + std::to_string(n) + " elements, got shape " + shape(t)};
  if (t.scalar_type() != at::kInt || t.device() != device)
    throw Raise{PyExc_TypeError, std::string(what) + " must be int32 on " + device.str() + ", got " + kind(t)};
  return t.stride(0) == 1 ? t : t.contiguous();
}

// a given output: like the query, contiguous rows that do not overlap
Tensor output(PyObject* o, const Tensor& q) {
  if (o == Py_None) return at::empty(q.sizes(), q.options());
  const Tensor& t = tensor(o, "out");
  if (t.sizes() != q.sizes() || t.scalar_type() != q.scalar_type() || t.device() != q.device() || t.stride(2) != 1)
    throw Raise{PyExc_ValueError, "out must be like the query, with contiguous rows"};
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes) throw Raise{PyExc_ValueError, "rows of out overlap"};
  return t;
}
float* lse_of(PyObject* o, const Tensor& q) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(o, "lse");
  if (t.dim() != 2 || t.size(0) != q.size(0) || t.size(1) != q.size(1) || t.scalar_type() != at::kFloat || !t.is_contiguous() ||
      t.device() != q.device())
    throw Raise{PyExc_ValueError, "lse must be a contiguous fp32 [rows, heads] tensor on the query's device"};
  return (float*)t.data_ptr();
}

void* stream_of(at::Device d) { return (void*)c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

// The cache as the C ABI wants it; `tuple` is (pages, dense_k, dense_v, w_sink, w_recent).
struct Cache {
  innerq_paged c{};
  at::ScalarType dtype;
  at::Device device{at::kCPU};
  Tensor table, slots, lens;

  explicit Cache(PyObject* tuple) {
    if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != 5) throw Raise{PyExc_TypeError, "not a cache"};
    const Tensor &pages = tensor(PyTuple_GET_ITEM(tuple, 0), "pages"), &k = tensor(PyTuple_GET_ITEM(tuple, 1), "dense_k"),
                 &v = tensor(PyTuple_GET_ITEM(tuple, 2), "dense_v");
    dtype = k.scalar_type();
    device = pages.device();
    c.struct_size = sizeof(c);
    c.dtype = dtype == at::kHalf ? INNERQ_DT_F16 : INNERQ_DT_BF16;
    c.D = kD;
    c.Hkv = k.size(1);
    c.page_tiles = pages.size(2);
    c.n_pages = pages.size(0);
    c.n_slots = k.size(0);
    c.w_sink = PyLong_AsLong(PyTuple_GET_ITEM(tuple, 3));
    c.w_recent = PyLong_AsLong(PyTuple_GET_ITEM(tuple, 4));
    c.pages = pages.data_ptr();
    c.dense_k = k.data_ptr();
    c.dense_v = v.data_ptr();
  }
  // the sequences of a call
  void batch(PyObject* t, PyObject* s, PyObject* n) {
    table = tensor(t, "page_table");
    if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != device)
      throw Raise{PyExc_TypeError, "page_table must be int32 [sequences, pages] on " + device.str()};
    if (table.size(1) > 1 && table.stride(1) != 1) table = table.contiguous();
    c.B = table.size(0);
    c.max_pages = table.size(1);
    slots = index(tensor(s, "slots"), "slots", c.B, device);
    lens = index(tensor(n, "seq_lens"), "seq_lens", c.B, device);
    c.table = (const int32_t*)table.data_ptr();
    c.table_stride = table.stride(0);
    c.slots = (const int32_t*)slots.data_ptr();
    c.seq_lens = (const int32_t*)lens.data_ptr();
  }
};

void check_cache(PyObject* const* a) {
  const Tensor &pages = tensor(a[0], "pages"), &k = tensor(a[1], "dense_k"), &v = tensor(a[2], "dense_v");
  const int64_t sink = integer(a[3], "w_sink"), recent = integer(a[4], "w_recent");
  need_cuda(pages, "pages");
  if (k.dim() != 4 || pages.dim() != 4)
    throw Raise{PyExc_ValueError, "pages " + shape(pages) + " and slots " + shape(k) + " must have four dimensions"};
  if (k.size(3) != kD) throw Raise{PyExc_NotImplementedError, "head_dim " + std::to_string(k.size(3)) + " is not built (128 is)"};
  if (sink < 0 || recent < 0 || sink % kTile || recent % kTile)
    throw Raise{PyExc_ValueError,
                "sink " + std::to_string(sink) + " and recent window " + std::to_string(recent) + " must be multiples of 32"};
  if (k.size(2) != sink + recent + kTile || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type())
    throw Raise{PyExc_ValueError, "slots must hold " + std::to_string(sink + recent + kTile) + " rows of keys and of values, got " +
                                      shape(k) + " and " + shape(v)};
  if (pages.scalar_type() != at::kByte || pages.size(1) != k.size(1) || pages.size(3) != kBlock)
    throw Raise{PyExc_ValueError, "pages must be uint8 [pages, " + std::to_string(k.size(1)) + ", tiles, 4608], got " +
                                      type_name(pages.scalar_type()) + " " + shape(pages)};
  if (!pages.is_contiguous() || !k.is_contiguous() || !v.is_contiguous())
    throw Raise{PyExc_ValueError, "pages and slots must be contiguous"};
  if (pages.device() != k.device() || pages.device() != v.device())
    throw Raise{PyExc_ValueError, "pages and slots must be on one device"};
  dtype_code(k.scalar_type());
}

// cos / sin: fp32 [positions, rot / 2], rows contiguous and 16-byte aligned
Tensor angles(PyObject* o, at::Device device) {
  const Tensor& t = tensor(o, "cos and sin");
  if (t.dim() != 2 || t.scalar_type() != at::kFloat || t.device() != device)
    throw Raise{PyExc_TypeError, "cos and sin must be fp32 [positions, rot / 2] on " + device.str()};
  if (t.stride(1) == 1 && t.stride(0) % 4 == 0 && (uintptr_t)t.data_ptr() % 16 == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// append(cache, q, k, v, page_table, slots, seq_lens, cu_seqlens, cos, sin, interleaved, return_k)
PyObject* append(PyObject* const* a) {
  Cache cache(a[0]);
  const at::ScalarType dtype = cache.dtype;
  const at::Device device = cache.device;
  const Tensor k = rows(tensor(a[2], "key"), "key", dtype, device), v = rows(tensor(a[3], "value"), "value", dtype, device);
  const int64_t T = k.size(0), hkv = cache.c.Hkv;
  if (k.size(1) != hkv || k.size(2) != kD || v.sizes() != k.sizes())
    throw Raise{PyExc_ValueError, "key " + shape(k) + " and value " + shape(v) + " must be [tokens, " + std::to_string(hkv) + ", 128]"};
  cache.batch(a[4], a[5], a[6]);
  innerq_paged_new n{};
  n.struct_size = sizeof(n);
  n.T = T;
  n.k = k.data_ptr();
  n.k_st = k.stride(0);
  n.k_sh = k.stride(1);
  n.v = v.data_ptr();
  n.v_st = v.stride(0);
  n.v_sh = v.stride(1);
  const c10::cuda::CUDAGuard guard(device);
  Tensor q, q_out, k_out, cu, cos, sin;
  if (a[1] != Py_None) {
    q = rows(tensor(a[1], "query"), "query", dtype, device);
    if (q.size(0) != T || q.size(2) != kD)
      throw Raise{PyExc_ValueError, "query " + shape(q) + " must be [" + std::to_string(T) + ", heads, 128]"};
    q_out = at::empty(q.sizes(), q.options());
    n.Hq = q.size(1);
    n.q = q.data_ptr();
    n.q_st = q.stride(0);
    n.q_sh = q.stride(1);
    n.q_out = q_out.data_ptr();
    n.qo_st = n.Hq * kD;
    n.qo_sh = kD;
  }
  if (a[7] != Py_None) {
    cu = index(tensor(a[7], "cu_seqlens"), "cu_seqlens", cache.c.B + 1, device);
    n.cu_seqlens = (const int32_t*)cu.data_ptr();
  } else if (T != cache.c.B) {
    throw Raise{PyExc_ValueError, std::to_string(T) + " tokens for " + std::to_string(cache.c.B) + " sequences need cu_seqlens"};
  }
  if ((a[8] == Py_None) != (a[9] == Py_None)) throw Raise{PyExc_ValueError, "cos and sin come together"};
  if (a[8] != Py_None) {
    cos = angles(a[8], device);
    sin = angles(a[9], device);
    if (cos.sizes() != sin.sizes()) throw Raise{PyExc_ValueError, "cos " + shape(cos) + " and sin " + shape(sin) + " differ"};
    if (cos.stride(0) != sin.stride(0)) {
      cos = cos.clone(at::MemoryFormat::Contiguous);
      sin = sin.clone(at::MemoryFormat::Contiguous);
    }
    n.rot_dim = 2 * cos.size(1);
    n.max_pos = cos.size(0);
    n.cs_stride = cos.stride(0);
    n.cos = (const float*)cos.data_ptr();
    n.sin = (const float*)sin.data_ptr();
    n.interleaved = truth(a[10]);
  }
  const bool return_k = truth(a[11]);
  if (return_k) {
    k_out = at::empty(k.sizes(), k.options());
    n.k_out = k_out.data_ptr();
    n.ko_st = hkv * kD;
    n.ko_sh = kD;
  }
  check(f_append(&cache.c, &n, stream_of(device)), "innerq_paged_append");
  PyObject* pq;
  if (q_out.defined()) {
    pq = THPVariable_Wrap(std::move(q_out));
  } else {
    Py_INCREF(Py_None);
    pq = Py_None;
  }
  if (!return_k) return pq;
  PyObject* pk = THPVariable_Wrap(std::move(k_out));
  PyObject* both = PyTuple_Pack(2, pq, pk);
  Py_DECREF(pq);
  Py_DECREF(pk);
  return both;
}

// attend(cache, q, page_table, slots, seq_lens, scale, out, lse)
PyObject* attend(PyObject* const* a) {
  Cache cache(a[0]);
  const Tensor q = rows(tensor(a[1], "query"), "query", cache.dtype, cache.device);
  cache.batch(a[2], a[3], a[4]);
  if (q.size(0) != cache.c.B || q.size(2) != kD)
    throw Raise{PyExc_ValueError, "query " + shape(q) + " must be [" + std::to_string(cache.c.B) + ", heads, 128]"};
  const float scale = scale_of(a[5]);
  const c10::cuda::CUDAGuard guard(cache.device);
  Tensor out = output(a[6], q);
  float* lse = lse_of(a[7], q);
  const int Hq = q.size(1);
  const int64_t bytes = f_workspace(&cache.c, Hq);
  if (bytes < 0) throw Failed{"innerq_paged_attn_workspace", Hq > 8 * cache.c.Hkv ? INNERQ_ERR_UNSUPPORTED : INNERQ_ERR_ARG};
  const Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));  // of this stream
  check(f_attn(&cache.c, Hq, q.data_ptr(), q.stride(0), q.stride(1), scale, ws.data_ptr(), bytes, out.data_ptr(), out.stride(0),
               out.stride(1), lse, stream_of(cache.device)),
        "innerq_paged_attn");
  return THPVariable_Wrap(std::move(out));
}

// read(cache, page_table, slots, seq_lens, starts, cu_seqlens, n_tokens)
PyObject* read(PyObject* const* a) {
  Cache cache(a[0]);
  cache.batch(a[1], a[2], a[3]);
  const Tensor starts = index(tensor(a[4], "starts"), "starts", cache.c.B, cache.device),
               cu = index(tensor(a[5], "cu_seqlens"), "cu_seqlens", cache.c.B + 1, cache.device);
  const int64_t n = integer(a[6], "n_tokens");
  if (n < 0 || n > 0x7fffffff) throw Raise{PyExc_ValueError, "n_tokens " + std::to_string(n)};
  const c10::cuda::CUDAGuard guard(cache.device);
  const auto options = at::TensorOptions().dtype(cache.dtype).device(cache.device);
  Tensor k = at::empty({n, cache.c.Hkv, kD}, options), v = at::empty({n, cache.c.Hkv, kD}, options);
  check(f_read(&cache.c, (const int32_t*)starts.data_ptr(), (const int32_t*)cu.data_ptr(), n, k.data_ptr(), v.data_ptr(),
               stream_of(cache.device)),
        "innerq_paged_read");
  PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v)), *both = PyTuple_Pack(2, pk, pv);
  Py_DECREF(pk);
  Py_DECREF(pv);
  return both;
}

// prompt(q, k, v, cu_seqlens, cu_seqlens_k, scale, causal, out, lse)
PyObject* prompt(PyObject* const* a) {
  const Tensor& q_in = tensor(a[0], "query");
  need_cuda(q_in, "query");
  const at::ScalarType dtype = q_in.scalar_type();
  const at::Device device = q_in.device();
  innerq_prompt_args p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_code(dtype);
  const Tensor q = rows(q_in, "query", dtype, device), k = rows(tensor(a[1], "key"), "key", dtype, device),
               v = rows(tensor(a[2], "value"), "value", dtype, device);
  if (k.sizes() != v.sizes() || k.size(2) != q.size(2))
    throw Raise{PyExc_ValueError, "shapes of query " + shape(q) + ", key " + shape(k) + " and value " + shape(v)};
  const Tensor cu = index(tensor(a[3], "cu_seqlens"), "cu_seqlens", -1, device);
  if (cu.size(0) < 1) throw Raise{PyExc_ValueError, "cu_seqlens must have at least one element"};
  const Tensor cu_k = a[4] == Py_None ? cu : index(tensor(a[4], "cu_seqlens_k"), "cu_seqlens_k", cu.size(0), device);
  p.scale = scale_of(a[5]);
  p.causal = truth(a[6]);
  const c10::cuda::CUDAGuard guard(device);
  const Tensor given = output(a[7], q);
  // rows that the kernel cannot write in 16-byte pieces: through a copy
  const bool fits = given.stride(0) % 8 == 0 && given.stride(1) % 8 == 0 && (uintptr_t)given.data_ptr() % 16 == 0;
  const Tensor out = fits ? given : given.clone(at::MemoryFormat::Contiguous);
  p.lse = lse_of(a[8], q);
  p.D = q.size(2);
  p.B = cu.size(0) - 1;
  p.Hq = q.size(1);
  p.Hkv = k.size(1);
  p.Tq = q.size(0);
  p.Tk = k.size(0);
  p.q = q.data_ptr();
  p.q_st = q.stride(0);
  p.q_sh = q.stride(1);
  p.k = k.data_ptr();
  p.k_st = k.stride(0);
  p.k_sh = k.stride(1);
  p.v = v.data_ptr();
  p.v_st = v.stride(0);
  p.v_sh = v.stride(1);
  p.cu_q = (const int32_t*)cu.data_ptr();
  p.cu_k = (const int32_t*)cu_k.data_ptr();
  p.out = out.data_ptr();
  p.o_st = out.stride(0);
  p.o_sh = out.stride(1);
  check(f_prompt(&p, stream_of(device)), "innerq_prompt_attn");
  if (!fits) given.copy_(out);
  return THPVariable_Wrap(given);
}

// ------------------------------------------------------------------ module ---
PyObject* raise(const Failed& f) {
  PyObject* lib = PyImport_ImportModule("innerq_b200._lib");
  PyObject* type = lib ? PyObject_GetAttrString(lib, "InnerqError") : nullptr;
  PyObject* e = type ? PyObject_CallFunction(type, "sis", f.fn, f.code, f_error()) : nullptr;
  if (e) PyErr_SetObject(type, e);
  Py_XDECREF(e);
  Py_XDECREF(type);
  Py_XDECREF(lib);
  return nullptr;
}

template <int N, PyObject* (*F)(PyObject* const*)>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments, got %zd", N, n);
    return nullptr;
  }
  if (!f_prompt) {
    PyErr_SetString(PyExc_RuntimeError, "bind() has not been called");
    return nullptr;
  }
  try {
    return F(a);
  } catch (const Raise& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const Failed& f) {
    return raise(f);
  } catch (const Pending&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    PyErr_SetString(type ? type : PyExc_MemoryError, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* check_entry(PyObject* const* a) {
  check_cache(a);
  Py_RETURN_NONE;
}

// bind(path): the library whose entry points are called
PyObject* bind(PyObject*, PyObject* arg) {
  const char* path = PyUnicode_AsUTF8(arg);
  if (!path) return nullptr;
  void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!h) {
    PyErr_SetString(PyExc_ImportError, dlerror());
    return nullptr;
  }
  f_append = (decltype(f_append))dlsym(h, "innerq_paged_append");
  f_read = (decltype(f_read))dlsym(h, "innerq_paged_read");
  f_workspace = (decltype(f_workspace))dlsym(h, "innerq_paged_attn_workspace");
  f_attn = (decltype(f_attn))dlsym(h, "innerq_paged_attn");
  f_error = (decltype(f_error))dlsym(h, "innerq_last_error");
  f_prompt = (decltype(f_prompt))dlsym(h, "innerq_prompt_attn");
  if (!f_append || !f_read || !f_workspace || !f_attn || !f_error || !f_prompt) {
    f_prompt = nullptr;
    PyErr_SetString(PyExc_ImportError, "the library lacks entry points of the paged cache; rebuild it");
    return nullptr;
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_O, "bind(path): the library whose entry points are called"},
    {"check_cache", (PyCFunction)(void*)entry<5, check_entry>, METH_FASTCALL, "check_cache(pages, dense_k, dense_v, w_sink, w_recent)"},
    {"append", (PyCFunction)(void*)entry<12, append>, METH_FASTCALL,
     "append(cache, q, k, v, page_table, slots, seq_lens, cu_seqlens, cos, sin, interleaved, return_k)"},
    {"attend", (PyCFunction)(void*)entry<8, attend>, METH_FASTCALL,
     "attend(cache, q, page_table, slots, seq_lens, scale, out, lse)"},
    {"read", (PyCFunction)(void*)entry<7, read>, METH_FASTCALL,
     "read(cache, page_table, slots, seq_lens, starts, cu_seqlens, n_tokens)"},
    {"prompt", (PyCFunction)(void*)entry<9, prompt>, METH_FASTCALL,
     "prompt(q, k, v, cu_seqlens, cu_seqlens_k, scale, causal, out, lse)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host side of the paged cache and of prompt attention.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
