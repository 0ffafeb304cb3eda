// Python binding of the paged-cache operators (paged.py): argument checks,
// output tensors and the C call in one step.  Their kernels run for 5 to 10 us
// in a decode step; the same host work in Python with ctypes took 13 to 24 us a
// call, here it takes 3 to 7 (reserve 17.3 -> 6.6, release 12.5 -> 4.2, append
// and read together 23.7 -> 7.6, attention 15 -> 4.3, 6.4 for blocks of query
// rows, which are two launches).  Nothing here touches
// the device but the C ABI, whose entries paged.py hands over (bind) from the
// library that it has loaded.
#include <Python.h>

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <cstdarg>

#include "../../include/dflash_b200.h"

namespace {

struct PyError {};   // a Python exception is set

[[noreturn]] void refuse(const char* fmt, ...) {
  char msg[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  PyErr_SetString(PyExc_ValueError, msg);
  throw PyError();
}

// ---- the library's entries
struct Lib {
  decltype(&dflash_paged_reserve_tracked) reserve;
  decltype(&dflash_paged_release) release;
  decltype(&dflash_paged_trim) trim;
  decltype(&dflash_q4_append) append;
  decltype(&dflash_q4_read) read;
  decltype(&dflash_q4_attention) attention;
  decltype(&dflash_last_error) last_error;
} lib;

void check(int status, const char* what) {
  if (status == DFLASH_OK) return;
  char why[1024] = "";
  lib.last_error(why, sizeof why);
  PyErr_Format(status == DFLASH_ERR_INVALID ? PyExc_ValueError : PyExc_RuntimeError, "%s failed: %s", what, why);
  throw PyError();
}

// ---- arguments
const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyError();
  return v;
}
int int32(PyObject* o, const char* name) {
  const long long v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s %lld is out of range", name, v);
  return (int)v;
}
bool boolean(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyError();
  return v != 0;
}
std::string describe(const at::Tensor& t) {
  std::ostringstream s;
  s << t.dtype() << " " << t.sizes() << " on " << t.device();
  return s.str();
}
int cuda_index(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("the paged cache's tensors must be on a CUDA device");
  return t.get_device();
}
// a contiguous int32 vector of n entries (any number if n < 0) on device dev
int32_t* i32(PyObject* o, const char* name, int64_t n, int dev, int64_t* count = nullptr) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev || t.dim() != 1 || !t.is_contiguous() ||
      (n >= 0 && t.numel() != n))
    refuse("%s must be a contiguous int32 vector%s on cuda:%d, got %s", name,
           n >= 0 ? (" of " + std::to_string(n)).c_str() : "", dev, describe(t).c_str());
  if (t.numel() > INT32_MAX) refuse("%s has more than 2^31 entries", name);
  if (count) *count = t.numel();
  return t.data_ptr<int32_t>();
}
int32_t* i32_or_none(PyObject* o, const char* name, int64_t n, int dev) { return o == Py_None ? nullptr : i32(o, name, n, dev); }
int32_t* status_of(PyObject* o, int dev) { return i32_or_none(o, "status", 1, dev); }

struct Table {
  int32_t* data;
  int64_t ld;
  int width;
};
Table table_of(PyObject* o, int64_t n, int dev) {
  const at::Tensor& t = tensor(o, "table");
  if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev || t.dim() != 2)
    refuse("table must be an int32 matrix [%lld, max_pages] on cuda:%d", (long long)n, dev);
  const int64_t width = t.size(1);
  if (t.size(0) != n || (t.stride(1) != 1 && width > 1) || width > INT32_MAX)
    refuse("table must be [%lld, max_pages] with contiguous rows, got %s", (long long)n, describe(t).c_str());
  return {t.data_ptr<int32_t>(), std::max(t.stride(0), width), (int)width};
}

struct Pool {
  uint8_t* data;
  int pages, nkv, page_size, dev;
};
Pool pool_of(PyObject* o) {
  const at::Tensor& t = tensor(o, "pool");
  const int dev = cuda_index(t);
  if (t.scalar_type() != at::kByte || t.dim() != 4 || !t.is_contiguous() || t.size(3) != 2304 || t.size(0) > INT32_MAX ||
      t.size(1) > INT32_MAX || t.size(2) > 4096)
    refuse("pool must be a contiguous uint8 tensor from q4_pool()");
  return {t.data_ptr<uint8_t>(), (int)t.size(0), (int)t.size(1), (int)t.size(2) * 16, dev};
}

// [rows, heads, 128] as the kernels can read it in whole 16 bytes: the tensor itself or a copy
struct Rows {
  at::Tensor t;
  const uint16_t* data;
  int64_t row, head;
  int rows, heads, bf16;
};
Rows rows_of(PyObject* o, const char* name, int64_t heads, int dev) {
  Rows r{tensor(o, name), nullptr, 0, 0, 0, 0, 0};
  const auto type = r.t.scalar_type();
  if ((type != at::kHalf && type != at::kBFloat16) || !r.t.is_cuda() || r.t.get_device() != dev || r.t.dim() != 3 ||
      r.t.size(2) != 128 || (heads >= 0 && r.t.size(1) != heads) || r.t.size(0) > INT32_MAX || r.t.size(1) > INT32_MAX)
    refuse("%s must be f16 or bf16 [rows, %s, 128] on cuda:%d, got %s", name,
           heads >= 0 ? std::to_string(heads).c_str() : "heads", dev, describe(r.t).c_str());
  if (r.t.stride(2) != 1 || (r.t.stride(0) | r.t.stride(1)) % 8 || reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16)
    r.t = r.t.clone(at::MemoryFormat::Contiguous);   // (contiguous() keeps a misaligned tensor, or a stride of one row)
  r.data = static_cast<const uint16_t*>(r.t.data_ptr());
  r.row = r.t.stride(0);
  r.head = r.t.stride(1);
  r.rows = (int)r.t.size(0);
  r.heads = (int)r.t.size(1);
  r.bf16 = type == at::kBFloat16;
  return r;
}

// ---- outputs
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int dev) {
  return at::empty(size, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)dev)));
}
// n entries of a vector from `at` on, as a tensor over the same storage
PyObject* slice(const at::Tensor& t, int64_t at, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(t.storage()), t.key_set(), t.dtype());
  impl->set_storage_offset(at);
  impl->set_sizes_contiguous({n});
  PyObject* o = THPVariable_Wrap(at::Tensor(std::move(impl)));
  if (!o) throw PyError();
  return o;
}
template <class... O>
PyObject* tuple(O... o) {
  PyObject* t = PyTuple_New(sizeof...(o));
  if (!t) throw PyError();
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(t, i++, o), ...);
  return t;
}

// the C call on the tensors' device and its current stream
template <class F, class... A>
void call(const char* what, F fn, int dev, A... a) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fn(a..., stream);
  Py_END_ALLOW_THREADS
  check(status, what);
}

template <PyObject* (*F)(PyObject* const*), int COUNT>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != COUNT) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", COUNT, n);
    return nullptr;
  }
  if (!lib.last_error) {
    PyErr_SetString(PyExc_RuntimeError, "bind() was not called");
    return nullptr;
  }
  try {
    return F(a);
  } catch (const PyError&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (lens, new_rows, pages, table, free_pages, head, page_size, num_slots, status, refused)
PyObject* reserve(PyObject* const* a) {
  const at::Tensor& lens = tensor(a[0], "lens");
  const int dev = cuda_index(lens);
  const int64_t n = lens.numel(), num_slots = int32(a[7], "num_slots");
  const int page_size = int32(a[6], "page_size");
  if (num_slots < 0) refuse("num_slots %lld", (long long)num_slots);
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[3], n, dev);
  int64_t num_pages;
  int32_t *l = i32(a[0], "lens", n, dev), *r = i32(a[1], "new_rows", n, dev), *p = i32(a[2], "pages", n, dev),
          *f = i32(a[4], "free_pages", -1, dev, &num_pages), *h = i32(a[5], "head", 1, dev), *s = status_of(a[8], dev),
          *refused = i32_or_none(a[9], "refused", n, dev);
  const at::Tensor out = empty({3 * n + 2 + num_slots}, at::kInt, dev);   // [starts | lens | pages | head | slots]
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_reserve", lib.reserve, dev, l, r, p, (int)n, page_size, t.data, t.ld, t.width, f, (int)num_pages, h, o,
       o + 3 * n + 2, (int)num_slots, o + n + 1, o + 2 * n + 1, o + 3 * n + 1, refused, s);
  return tuple(slice(out, 0, n + 1), slice(out, 3 * n + 2, num_slots), slice(out, n + 1, n), slice(out, 2 * n + 1, n),
               slice(out, 3 * n + 1, 1));
}

// (keep, pages, table, free_pages, head, page_size, status)
PyObject* release(PyObject* const* a) {
  const at::Tensor& keep = tensor(a[0], "keep");
  const int dev = cuda_index(keep);
  const int64_t n = keep.numel();
  const int page_size = int32(a[5], "page_size");
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[2], n, dev);
  int64_t num_pages;
  int32_t *k = i32(a[0], "keep", n, dev), *p = i32(a[1], "pages", n, dev),
          *f = i32(a[3], "free_pages", -1, dev, &num_pages), *h = i32(a[4], "head", 1, dev), *s = status_of(a[6], dev);
  const at::Tensor out = empty({n + 1}, at::kInt, dev);
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_release", lib.release, dev, k, p, (int)n, page_size, t.data, t.ld, t.width, f, (int)num_pages, h, o,
       o + n, s);
  return tuple(slice(out, 0, n), slice(out, n, 1));
}

// (lens, counts: a tensor or a number, refused, out: or None) -> out
PyObject* trim(PyObject* const* a) {
  const at::Tensor& lens = tensor(a[0], "lens");
  const int dev = cuda_index(lens);
  const int64_t n = lens.numel();
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const int32_t* l = i32(a[0], "lens", n, dev);
  const int32_t* counts = PyLong_Check(a[1]) ? nullptr : i32(a[1], "counts", n, dev);
  const int count = counts ? 0 : int32(a[1], "count");
  const int32_t* refused = i32_or_none(a[2], "refused", n, dev);
  const at::Tensor out = a[3] == Py_None ? empty({n}, at::kInt, dev) : tensor(a[3], "out");
  int32_t* o = a[3] == Py_None ? out.data_ptr<int32_t>() : i32(a[3], "out", n, dev);
  call("dflash_paged_trim", lib.trim, dev, l, counts, count, refused, (int)n, o);
  return a[3] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[3]);
}

// (k, v, slots, pool, status)
PyObject* append(PyObject* const* a) {
  const Pool p = pool_of(a[3]);
  const Rows k = rows_of(a[0], "k", p.nkv, p.dev), v = rows_of(a[1], "v", p.nkv, p.dev);
  if (k.bf16 != v.bf16 || k.rows != v.rows) refuse("k and v must have the same type and number of rows");
  call("dflash_q4_append", lib.append, p.dev, k.data, k.row, k.head, v.data, v.row, v.head, k.bf16,
       i32(a[2], "slots", k.rows, p.dev), k.rows, p.nkv, p.data, p.pages, p.page_size, status_of(a[4], p.dev));
  Py_RETURN_NONE;
}

// (pool, slots, bf16)
PyObject* read(PyObject* const* a) {
  const Pool p = pool_of(a[0]);
  const bool bf16 = boolean(a[2]);
  int64_t rows;
  const int32_t* slots = i32(a[1], "slots", -1, p.dev, &rows);
  const at::Tensor k = empty({rows, p.nkv, 128}, bf16 ? at::kBFloat16 : at::kHalf, p.dev), v = at::empty_like(k);
  call("dflash_q4_read", lib.read, p.dev, p.data, p.pages, p.page_size, slots, (int)rows, p.nkv, (int)bf16,
       static_cast<uint16_t*>(k.data_ptr()), static_cast<uint16_t*>(v.data_ptr()));
  return tuple(THPVariable_Wrap(k), THPVariable_Wrap(v));
}

// (q, pool, table, lens, starts, max_rows, causal, sink, window, scale, out, status, workspace)
PyObject* attention(PyObject* const* a) {
  const Pool p = pool_of(a[1]);
  const Rows q = rows_of(a[0], "q", -1, p.dev);
  int64_t n;
  const int32_t* lens = i32(a[3], "lens", -1, p.dev, &n);
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[2], n, p.dev);
  const int32_t* starts = a[4] == Py_None ? nullptr : i32(a[4], "starts", n + 1, p.dev);
  const double scale = PyFloat_AsDouble(a[9]);
  if (scale == -1.0 && PyErr_Occurred()) throw PyError();
  at::Tensor out;
  if (a[10] == Py_None) {
    out = empty(q.t.sizes(), q.t.scalar_type(), p.dev);
  } else {
    out = tensor(a[10], "out");
    if (!out.sizes().equals(q.t.sizes()) || out.scalar_type() != q.t.scalar_type() || !out.is_cuda() ||
        out.get_device() != p.dev || !out.is_contiguous())
      refuse("out must be contiguous, of q's shape, type and device");
  }
  const at::Tensor& ws = tensor(a[12], "workspace");
  if (!ws.is_cuda() || ws.get_device() != p.dev || !ws.is_contiguous()) refuse("workspace must be on cuda:%d", p.dev);
  call("dflash_q4_attention", lib.attention, p.dev, q.data, q.row, q.head, q.bf16, p.data, p.pages, p.page_size, t.data, t.ld,
       t.width, lens, starts, (int)n, q.rows, int32(a[5], "max_rows"), q.heads, p.nkv, (int)boolean(a[6]),
       int32(a[7], "sink"), int32(a[8], "window"), (float)scale, static_cast<uint16_t*>(out.data_ptr()),
       status_of(a[11], p.dev), ws.data_ptr(), (size_t)ws.nbytes());
  return a[10] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[10]);
}

// (device) -> whether its current stream is being captured
PyObject* capturing(PyObject* const* a) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)int32(a[0], "device"));
  return PyBool_FromLong(c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None);
}

// addresses of the library's entries, in the order of Lib
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* at[7];
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind: 7 addresses expected");
    return nullptr;
  }
  for (int i = 0; i < 7; ++i)
    if (!(at[i] = PyLong_AsVoidPtr(a[i]))) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: NULL");
      return nullptr;
    }
  lib.reserve = reinterpret_cast<decltype(lib.reserve)>(at[0]);
  lib.release = reinterpret_cast<decltype(lib.release)>(at[1]);
  lib.trim = reinterpret_cast<decltype(lib.trim)>(at[2]);
  lib.append = reinterpret_cast<decltype(lib.append)>(at[3]);
  lib.read = reinterpret_cast<decltype(lib.read)>(at[4]);
  lib.attention = reinterpret_cast<decltype(lib.attention)>(at[5]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[6]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), int COUNT>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<F, COUNT>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    method<reserve, 10>("reserve"),
    method<release, 7>("release"),
    method<trim, 4>("trim"),
    method<capturing, 1>("capturing"),
    method<append, 5>("append"),
    method<read, 3>("read"),
    method<attention, 13>("attention"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "dflash_paged", "Paged 4-bit cache operators (see paged.py).", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dflash_paged() { return PyModule_Create(&module); }
