// Host binding of the 8-bit cache and the windowed attention: checks the tensors of a call and hands
// their addresses to the C entry points (include/paged_evict.h) on the current stream of their device.
//
// These calls are issued once per layer and step; the smallest of them keep the GPU busy for 5 us.
// Checked and converted in Python (ctypes) they cost 11 us of host time per call besides the launch,
// here under 1 us, so a small batch is bound by the GPU and not by the interpreter.
// The functions take positional arguments only; ops.py gives them names, defaults and documentation.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <string>

#include "../../include/paged_evict.h"

namespace {

struct PyFail {};  // a Python exception is set

#define REQ(cond, exc, ...)           \
  do {                                \
    if (!(cond)) {                    \
      PyErr_Format((exc), __VA_ARGS__); \
      throw PyFail{};                 \
    }                                 \
  } while (0)

const at::Tensor& tensor(const char* what, const char* name, PyObject* o) {
  REQ(THPVariable_Check(o), PyExc_TypeError, "%s: %s must be a tensor", what, name);
  return THPVariable_Unpack(o);
}

int integer(const char* what, const char* name, PyObject* o) {
  PyObject* i = PyNumber_Index(o);
  if (i == nullptr) throw PyFail{};
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw PyFail{};
  REQ(v >= INT_MIN && v <= INT_MAX, PyExc_ValueError, "%s: %s does not fit 32 bits", what, name);
  return (int)v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFail{};
  return v;
}

int row_dtype(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PE_BF16;
    case at::kHalf: return PE_F16;
    default: return -1;
  }
}

int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }

// [rows, heads, head_size] whose rows are dense and 16-byte aligned
void check_rows(const char* what, const char* name, const at::Tensor& t, int64_t heads, int64_t head_size) {
  REQ(t.dim() == 3 && t.size(1) == heads && t.size(2) == head_size, PyExc_RuntimeError,
      "%s: %s must be [rows, %lld, %lld]", what, name, (long long)heads, (long long)head_size);
  if (t.numel() == 0) return;
  REQ(t.stride(2) == 1 && (heads == 1 || t.stride(1) == head_size), PyExc_RuntimeError,
      "%s: the rows of %s must be dense", what, name);
  // a tensor of one row is never stepped over: any row stride will do
  REQ((uintptr_t)t.data_ptr() % 16 == 0 && (t.size(0) == 1 || t.stride(0) % 8 == 0), PyExc_RuntimeError,
      "%s: the rows of %s must be 16-byte aligned", what, name);
}

// all tensors on one GPU; its index
int device_of(std::initializer_list<const at::Tensor*> ts) {
  int dev = -1;
  for (const at::Tensor* t : ts) {
    if (t == nullptr) continue;
    REQ(t->is_cuda(), PyExc_RuntimeError,
        "paged_evict ops run on the GPU only (got a %s tensor); there is no CPU fallback",
        c10::DeviceTypeName(t->device().type(), true).c_str());
    const int d = t->get_device();
    REQ(dev < 0 || dev == d, PyExc_RuntimeError, "paged_evict: tensors on different devices");
    dev = d;
  }
  return dev;
}

struct Paged {
  const at::Tensor &k, &v, &tables, &lens;
  int64_t nb, H, D, bs, S;
  int fmt = PE_KV_SAME;
};

Paged check_paged(const char* what, PyObject* kc, PyObject* vc, PyObject* tb, PyObject* ln, int64_t x) {
  Paged p{tensor(what, "key_cache", kc), tensor(what, "value_cache", vc), tensor(what, "block_tables", tb),
          tensor(what, "seq_lens", ln), 0, 0, 0, 0, 0};
  REQ(p.k.dim() == 5 && p.v.dim() == 4, PyExc_RuntimeError, "%s: key_cache must be 5-d and value_cache 4-d", what);
  p.nb = p.v.size(0), p.H = p.v.size(1), p.D = p.v.size(2), p.bs = p.v.size(3);
  REQ(p.nb > 0 && p.H > 0 && p.D > 0 && p.bs > 0 && p.D % x == 0 && p.k.size(0) == p.nb && p.k.size(1) == p.H &&
          p.k.size(2) == p.D / x && p.k.size(3) == p.bs && p.k.size(4) == x,
      PyExc_RuntimeError, "%s: key_cache must be [%lld, %lld, %lld/%lld, %lld, %lld]", what, (long long)p.nb,
      (long long)p.H, (long long)p.D, (long long)x, (long long)p.bs, (long long)x);
  REQ(p.k.scalar_type() == p.v.scalar_type(), PyExc_RuntimeError, "%s: key and value cache differ in dtype", what);
  REQ(p.k.is_contiguous() && p.v.is_contiguous(), PyExc_RuntimeError, "%s: caches must be contiguous", what);
  REQ(p.tables.scalar_type() == at::kInt && p.lens.scalar_type() == at::kInt, PyExc_RuntimeError,
      "%s: block_tables and seq_lens must be int32", what);
  REQ(p.tables.dim() == 2 && p.tables.is_contiguous(), PyExc_RuntimeError,
      "%s: block_tables must be contiguous [num_seqs, max_blocks]", what);
  p.S = p.tables.size(0);
  REQ(p.lens.dim() == 1 && p.lens.size(0) == p.S && p.lens.is_contiguous(), PyExc_RuntimeError,
      "%s: seq_lens must be contiguous [num_seqs]", what);
  REQ(p.nb <= INT_MAX && p.S <= INT_MAX && p.tables.size(1) <= INT_MAX, PyExc_RuntimeError, "%s: too many blocks", what);
  return p;
}

Paged check_8bit(const char* what, PyObject* kc, PyObject* vc, const at::Tensor& scales, PyObject* tb,
                 PyObject* ln, PyObject* format, const at::Tensor& rows) {
  const char* f = PyUnicode_Check(format) ? PyUnicode_AsUTF8(format) : nullptr;
  const std::string name = f ? f : "";
  const int fmt = name == "fp8" || name == "fp8_e4m3" ? PE_KV_FP8_E4M3 : name == "int8" ? PE_KV_INT8 : PE_KV_SAME;
  REQ(fmt != PE_KV_SAME, PyExc_ValueError, "%s: kv_cache_dtype must be one of 'fp8', 'fp8_e4m3', 'int8', got %R",
      what, format);
  const at::ScalarType st = tensor(what, "key_cache", kc).scalar_type();
  if (fmt == PE_KV_INT8)
    REQ(st == at::kChar, PyExc_RuntimeError, "%s: an int8 cache is held in torch.int8", what);
  else
    REQ(st == at::kFloat8_e4m3fn || st == at::kByte, PyExc_RuntimeError,
        "%s: an fp8 cache is held in torch.float8_e4m3fn or torch.uint8", what);
  REQ(row_dtype(rows) >= 0, PyExc_RuntimeError, "%s: bfloat16 or float16 rows expected", what);
  Paged p = check_paged(what, kc, vc, tb, ln, 16);
  p.fmt = fmt;
  REQ(scales.scalar_type() == at::kFloat && scales.dim() == 3 && scales.size(0) == p.nb && scales.size(1) == p.H &&
          scales.size(2) == 2 && scales.is_contiguous(),
      PyExc_RuntimeError, "%s: kv_scales must be contiguous float32 [%lld, %lld, 2]", what, (long long)p.nb,
      (long long)p.H);
  return p;
}

void check_new_rows(const char* what, const at::Tensor& k, const at::Tensor& v, const Paged& p) {
  check_rows(what, "key", k, p.H, p.D);
  check_rows(what, "value", v, p.H, p.D);
  REQ(k.size(0) == v.size(0) && k.scalar_type() == v.scalar_type(), PyExc_RuntimeError,
      "%s: key and value differ in shape or dtype", what);
}

void check_decode(const char* what, const at::Tensor& out, const at::Tensor& q, int kv_heads, int block_size,
                  const Paged& p, int window, int sinks) {
  REQ(kv_heads == p.H && block_size == p.bs, PyExc_RuntimeError,
      "%s: cache shape does not match num_kv_heads/block_size", what);
  REQ(q.dim() == 3 && q.size(0) == p.S && q.size(1) > 0 && q.size(1) % p.H == 0, PyExc_RuntimeError,
      "%s: query must be [num_seqs, num_heads, head_size] with num_heads a multiple of num_kv_heads", what);
  check_rows(what, "query", q, q.size(1), p.D);
  REQ(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous(), PyExc_RuntimeError,
      "%s: out must be contiguous, of query's shape and dtype", what);
  REQ(window >= 0 && sinks >= 0, PyExc_ValueError, "%s: sliding_window and num_sinks must not be negative", what);
}

struct WithoutGil {  // (restored before an exception reaches the caller)
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// runs `fn` (stream) -> status with device `dev` current
template <typename F>
void launch(const char* what, int dev, F&& fn) {
  int rc;
  {
    const WithoutGil free;
    const c10::hip::HIPGuard guard((c10::DeviceIndex)dev);
    rc = fn((void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream());
  }
  REQ(rc == 0, PyExc_RuntimeError, "paged_evict %s failed (status %d): %s", what, rc, pe_last_error());
}

// Split-KV partials of one call: a buffer of its own from torch's allocator, so that calls on two
// streams, or in two captured graphs, never share one
struct Workspace {
  at::Tensor t;
  void* p = nullptr;
  int64_t bytes = 0;
  Workspace(const Paged& c, const at::Tensor& q, int max_len, int window, int sinks) {
    bytes = pe_paged_window_workspace_bytes((int)c.S, (int)q.size(1), (int)c.H, (int)c.D, max_len, window, sinks, c.fmt);
    if (bytes > 0) {
      t = at::empty({bytes}, q.options().dtype(at::kByte));
      p = t.data_ptr();
    }
  }
};

PyObject* none() { Py_RETURN_NONE; }

template <typename F>
PyObject* guarded(const char* what, Py_ssize_t n, Py_ssize_t want, F&& body) {
  try {
    REQ(n == want, PyExc_TypeError, "%s: %zd arguments expected, got %zd", what, want, n);
    return body();
  } catch (const PyFail&) {
  } catch (const c10::OutOfMemoryError& e) {  // (as torch's own allocations raise it)
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* reshape_and_cache_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "reshape_and_cache_8bit";
  return guarded(what, n, 10, [&] {
    const at::Tensor &k = tensor(what, "key", a[0]), &v = tensor(what, "value", a[1]), &sc = tensor(what, "kv_scales", a[4]);
    const Paged p = check_8bit(what, a[2], a[3], sc, a[5], a[6], a[9], k);
    check_new_rows(what, k, v, p);
    const at::Tensor* cu = a[7] == Py_None ? nullptr : &tensor(what, "cu_q", a[7]);
    if (cu == nullptr)
      REQ(k.size(0) == p.S, PyExc_RuntimeError, "%s: without cu_q key/value hold one row per sequence", what);
    else
      REQ(cu->scalar_type() == at::kInt && cu->dim() == 1 && cu->size(0) == p.S + 1 && cu->is_contiguous(),
          PyExc_RuntimeError, "%s: cu_q must be contiguous int32 [num_seqs + 1]", what);
    const int max_q = integer(what, "max_q_len", a[8]);
    REQ(max_q >= 0, PyExc_ValueError, "%s: negative max_q_len", what);
    const int dev = device_of({&k, &v, &p.k, &p.v, &sc, &p.tables, &p.lens, cu});
    if (p.S == 0 || k.size(0) == 0) return none();
    launch(what, dev, [&](void* st) {
      return pe_reshape_and_cache_8bit(k.data_ptr(), v.data_ptr(), p.k.data_ptr(), p.v.data_ptr(),
                                       (float*)sc.data_ptr(), (const int32_t*)p.tables.data_ptr(),
                                       (const int32_t*)p.lens.data_ptr(), cu ? (const int32_t*)cu->data_ptr() : nullptr,
                                       (int)p.S, k.size(0), max_q, row_stride(k), row_stride(v), (int)p.H, (int)p.D,
                                       (int)p.bs, p.nb, (int)p.tables.size(1), p.H * p.D * p.bs, p.D * p.bs,
                                       row_dtype(k), p.fmt, st);
    });
    return none();
  });
}

PyObject* paged_attention_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "paged_attention_8bit";
  return guarded(what, n, 14, [&] {
    const at::Tensor &out = tensor(what, "out", a[0]), &q = tensor(what, "query", a[1]), &sc = tensor(what, "kv_scales", a[4]);
    const Paged p = check_8bit(what, a[2], a[3], sc, a[7], a[8], a[11], q);
    const double scale = real(a[6]);
    const int max_len = integer(what, "max_seq_len", a[10]), window = integer(what, "sliding_window", a[12]),
              sinks = integer(what, "num_sinks", a[13]);
    check_decode(what, out, q, integer(what, "num_kv_heads", a[5]), integer(what, "block_size", a[9]), p, window, sinks);
    const int dev = device_of({&out, &q, &p.k, &p.v, &sc, &p.tables, &p.lens});
    if (p.S == 0) return none();
    const Workspace ws(p, q, max_len, window, sinks);
    launch(what, dev, [&](void* st) {
      return pe_paged_decode_8bit(out.data_ptr(), q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(),
                                  (const float*)sc.data_ptr(), (const int32_t*)p.tables.data_ptr(),
                                  (const int32_t*)p.lens.data_ptr(), (int)p.S, (int)q.size(1), (int)p.H, (int)p.D,
                                  (int)p.bs, p.nb, (int)p.tables.size(1), row_stride(q), p.H * p.D * p.bs, p.D * p.bs,
                                  (float)scale, max_len, window, sinks, row_dtype(q), p.fmt, ws.p, ws.bytes, st);
    });
    return none();
  });
}

PyObject* decode_step_8bit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "decode_step_8bit";
  return guarded(what, n, 16, [&] {
    const at::Tensor &out = tensor(what, "out", a[0]), &q = tensor(what, "query", a[1]), &k = tensor(what, "key", a[2]),
                     &v = tensor(what, "value", a[3]), &sc = tensor(what, "kv_scales", a[6]);
    const Paged p = check_8bit(what, a[4], a[5], sc, a[9], a[10], a[13], q);
    const double scale = real(a[8]);
    const int max_len = integer(what, "max_seq_len", a[12]), window = integer(what, "sliding_window", a[14]),
              sinks = integer(what, "num_sinks", a[15]);
    check_decode(what, out, q, integer(what, "num_kv_heads", a[7]), integer(what, "block_size", a[11]), p, window, sinks);
    check_new_rows(what, k, v, p);
    REQ(k.size(0) == p.S && k.scalar_type() == q.scalar_type(), PyExc_RuntimeError,
        "%s: key/value must be [num_seqs, num_kv_heads, head_size] of query's dtype", what);
    const int dev = device_of({&out, &q, &k, &v, &p.k, &p.v, &sc, &p.tables, &p.lens});
    if (p.S == 0) return none();
    const Workspace ws(p, q, max_len, window, sinks);
    launch(what, dev, [&](void* st) {
      return pe_decode_step_8bit(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), p.k.data_ptr(),
                                 p.v.data_ptr(), (float*)sc.data_ptr(), (const int32_t*)p.tables.data_ptr(),
                                 (const int32_t*)p.lens.data_ptr(), (int)p.S, (int)q.size(1), (int)p.H, (int)p.D,
                                 (int)p.bs, p.nb, (int)p.tables.size(1), row_stride(q), row_stride(k), row_stride(v),
                                 p.H * p.D * p.bs, p.D * p.bs, (float)scale, max_len, window, sinks, row_dtype(q),
                                 p.fmt, ws.p, ws.bytes, st);
    });
    return none();
  });
}

PyObject* paged_attention_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "paged_attention_window";
  return guarded(what, n, 12, [&] {
    const at::Tensor &out = tensor(what, "out", a[0]), &q = tensor(what, "query", a[1]);
    REQ(row_dtype(q) >= 0 && tensor(what, "key_cache", a[2]).scalar_type() == q.scalar_type(), PyExc_RuntimeError,
        "%s: query and caches must share bfloat16 or float16", what);
    const Paged p = check_paged(what, a[2], a[3], a[6], a[7], 8);
    const double scale = real(a[5]);
    const int max_len = integer(what, "max_seq_len", a[9]), window = integer(what, "sliding_window", a[10]),
              sinks = integer(what, "num_sinks", a[11]);
    check_decode(what, out, q, integer(what, "num_kv_heads", a[4]), integer(what, "block_size", a[8]), p, window, sinks);
    const int dev = device_of({&out, &q, &p.k, &p.v, &p.tables, &p.lens});
    if (p.S == 0) return none();
    const Workspace ws(p, q, max_len, window, sinks);
    launch(what, dev, [&](void* st) {
      return pe_paged_decode_window(out.data_ptr(), q.data_ptr(), p.k.data_ptr(), p.v.data_ptr(),
                                    (const int32_t*)p.tables.data_ptr(), (const int32_t*)p.lens.data_ptr(), (int)p.S,
                                    (int)q.size(1), (int)p.H, (int)p.D, (int)p.bs, p.nb, (int)p.tables.size(1),
                                    row_stride(q), p.H * p.D * p.bs, p.D * p.bs, (float)scale, max_len, window, sinks,
                                    row_dtype(q), ws.p, ws.bytes, st);
    });
    return none();
  });
}

PyObject* prefill_window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const char* what = "prefill_window";
  return guarded(what, n, 10, [&]() -> PyObject* {
    const at::Tensor &q = tensor(what, "query", a[0]), &k = tensor(what, "key", a[1]), &v = tensor(what, "value", a[2]),
                     &cu_q = tensor(what, "cu_q", a[3]), &cu_kv = tensor(what, "cu_kv", a[4]);
    REQ(q.dim() == 3 && k.dim() == 3 && k.size(1) > 0 && q.size(1) > 0 && q.size(1) % k.size(1) == 0 &&
            v.sizes() == k.sizes(),
        PyExc_RuntimeError, "%s: query [Tq, Hq, D], key/value [Tkv, Hkv, D] expected, Hq a multiple of Hkv", what);
    REQ(row_dtype(q) >= 0 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
        PyExc_RuntimeError, "%s: query, key and value must share bfloat16 or float16", what);
    const int64_t Hq = q.size(1), H = k.size(1), D = q.size(2);
    check_rows(what, "query", q, Hq, D);
    check_rows(what, "key", k, H, D);
    check_rows(what, "value", v, H, D);
    for (const at::Tensor* t : {&cu_q, &cu_kv})
      REQ(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) >= 1 && t->size(0) == cu_q.size(0) &&
              t->size(0) <= INT_MAX && t->is_contiguous(),
          PyExc_RuntimeError, "%s: cu_q/cu_kv must be contiguous int32 [num_requests + 1]", what);
    const int max_q = integer(what, "max_q_len", a[5]), window = integer(what, "sliding_window", a[7]),
              sinks = integer(what, "num_sinks", a[8]);
    const double scale = real(a[6]);
    REQ(window >= 0 && sinks >= 0 && max_q >= 0, PyExc_ValueError,
        "%s: max_q_len, sliding_window and num_sinks must not be negative", what);
    at::Tensor out;
    if (a[9] != Py_None) {
      out = tensor(what, "out", a[9]);
      check_rows(what, "out", out, Hq, D);
      REQ(out.size(0) == q.size(0) && out.scalar_type() == q.scalar_type(), PyExc_RuntimeError,
          "%s: out must have query's shape and dtype", what);
    }
    const int dev = device_of({&q, &k, &v, &cu_q, &cu_kv, out.defined() ? &out : nullptr});
    const bool any = q.size(0) > 0 && cu_q.size(0) > 1 && max_q > 0;
    // (a fresh output is zero where there is nothing to attend)
    if (!out.defined())
      out = any && k.size(0) > 0 ? at::empty({q.size(0), Hq, D}, q.options()) : at::zeros({q.size(0), Hq, D}, q.options());
    if (any) {  // (without kv rows too: the kernel writes the zeros of the requests' rows)
      launch(what, dev, [&](void* st) {
        return pe_prefill_window(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 (const int32_t*)cu_q.data_ptr(), (const int32_t*)cu_kv.data_ptr(),
                                 (int)cu_q.size(0) - 1, max_q, q.size(0), k.size(0), (int)Hq, (int)H, (int)D, row_stride(q), row_stride(k),
                                 row_stride(v), row_stride(out), (float)scale, window, sinks, row_dtype(q), st);
      });
    }
    return THPVariable_Wrap(out);
  });
}

#define METHOD(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(reshape_and_cache_8bit), METHOD(paged_attention_8bit), METHOD(decode_step_8bit),
                         METHOD(paged_attention_window), METHOD(prefill_window), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host binding of libpaged_evict.so", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
