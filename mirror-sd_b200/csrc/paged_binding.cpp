// Python binding of the paged-cache operators (paged.py) and of those around a
// decode step (rope.py, sampling.py): argument checks,
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
#include <cstring>

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
  decltype(&dflash_paged_fork) fork;
  decltype(&dflash_paged_reserve_forked) reserve_forked;
  decltype(&dflash_paged_release_forked) release_forked;
  decltype(&dflash_q4_copy_pages) copy_pages;
  decltype(&dflash_paged_prefix_plan) prefix_plan;
  decltype(&dflash_q4_prefix_attention) prefix_attention;
  decltype(&dflash_rope) rope;
  decltype(&dflash_verify_drafts) verify;
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

at::Tensor output_like(PyObject* o, const at::Tensor& q, int dev) {   // a new tensor for None
  if (o == Py_None) return empty(q.sizes(), q.scalar_type(), dev);
  const at::Tensor& out = tensor(o, "out");
  if (!out.sizes().equals(q.sizes()) || out.scalar_type() != q.scalar_type() || !out.is_cuda() || out.get_device() != dev ||
      !out.is_contiguous())
    refuse("out must be contiguous, of q's shape, type and device");
  return out;
}
const at::Tensor& workspace_of(PyObject* o, int dev) {
  const at::Tensor& ws = tensor(o, "workspace");
  if (!ws.is_cuda() || ws.get_device() != dev || !ws.is_contiguous()) refuse("workspace must be on cuda:%d", dev);
  return ws;
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
  const at::Tensor out = output_like(a[10], q.t, p.dev);
  const at::Tensor& ws = workspace_of(a[12], p.dev);
  call("dflash_q4_attention", lib.attention, p.dev, q.data, q.row, q.head, q.bf16, p.data, p.pages, p.page_size, t.data, t.ld,
       t.width, lens, starts, (int)n, q.rows, int32(a[5], "max_rows"), q.heads, p.nkv, (int)boolean(a[6]),
       int32(a[7], "sink"), int32(a[8], "window"), (float)scale, static_cast<uint16_t*>(out.data_ptr()),
       status_of(a[11], p.dev), ws.data_ptr(), (size_t)ws.nbytes());
  return a[10] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[10]);
}

// (table, lens, starts, max_rows, page_size, groups, causal, least) -> (group_starts, prefix, row_of, skip, own_lens)
PyObject* prefix_plan(PyObject* const* a) {
  const at::Tensor& lens = tensor(a[1], "lens");
  const int dev = cuda_index(lens);
  const int64_t n = lens.numel();
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[0], n, dev);
  const int32_t *l = i32(a[1], "lens", n, dev), *starts = a[2] == Py_None ? nullptr : i32(a[2], "starts", n + 1, dev);
  int64_t bounds;
  const int32_t* groups = i32(a[5], "groups", -1, dev, &bounds);
  const int64_t g = bounds - 1;
  if (g < 1 || g > DFLASH_PAGED_MAX_SEQS) refuse("%lld groups outside [1, %d]", (long long)g, DFLASH_PAGED_MAX_SEQS);
  const at::Tensor out = empty({3 * g + 1 + 2 * n}, at::kInt, dev);   // [group_starts | prefix | row_of | skip | own_lens]
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_prefix_plan", lib.prefix_plan, dev, t.data, t.ld, t.width, l, starts, (int)n, int32(a[3], "max_rows"),
       int32(a[4], "page_size"), groups, (int)g, (int)boolean(a[6]), (int64_t)integer(a[7]), o, o + g + 1, o + 2 * g + 1, o + 3 * g + 1, o + 3 * g + 1 + n);
  return tuple(slice(out, 0, g + 1), slice(out, g + 1, g), slice(out, 2 * g + 1, g), slice(out, 3 * g + 1, n),
               slice(out, 3 * g + 1 + n, n));
}

// (q, pool, table, starts, max_rows, group_starts, prefix, row_of, max_group, skip, own_lens, causal, scale, out, status, workspace)
PyObject* prefix_attention(PyObject* const* a) {
  const Pool p = pool_of(a[1]);
  const Rows q = rows_of(a[0], "q", -1, p.dev);
  int64_t n, g;
  const int32_t* own_lens = i32(a[10], "own_lens", -1, p.dev, &n);
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[2], n, p.dev);
  const int32_t* starts = a[3] == Py_None ? nullptr : i32(a[3], "starts", n + 1, p.dev);
  const int32_t* prefix = i32(a[6], "prefix", -1, p.dev, &g);
  const int32_t *group_starts = i32(a[5], "group_starts", g + 1, p.dev), *row_of = i32(a[7], "row_of", g, p.dev),
                *skip = i32(a[9], "skip", n, p.dev);
  const double scale = PyFloat_AsDouble(a[12]);
  if (scale == -1.0 && PyErr_Occurred()) throw PyError();
  const at::Tensor out = output_like(a[13], q.t, p.dev);
  const at::Tensor& ws = workspace_of(a[15], p.dev);
  call("dflash_q4_prefix_attention", lib.prefix_attention, p.dev, q.data, q.row, q.head, q.bf16, p.data, p.pages, p.page_size,
       t.data, t.ld, t.width, starts, (int)n, q.rows, int32(a[4], "max_rows"), group_starts, prefix, row_of, (int)g,
       int32(a[8], "max_group"), skip, own_lens, q.heads, p.nkv, (int)boolean(a[11]), (float)scale,
       static_cast<uint16_t*>(out.data_ptr()), status_of(a[14], p.dev), ws.data_ptr(), (size_t)ws.nbytes());
  return a[13] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[13]);
}

// (device) -> whether its current stream is being captured
PyObject* capturing(PyObject* const* a) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)int32(a[0], "device"));
  return PyBool_FromLong(c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None);
}

// ---- pages that several requests hold
int32_t* holders_of(PyObject* o, int64_t num_pages, int dev) {
  const at::Tensor& t = tensor(o, "holders");
  if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != dev || t.dim() != 2 || t.size(0) != 2 ||
      (num_pages >= 0 && t.size(1) != num_pages) || t.size(1) > INT32_MAX || !t.is_contiguous())
    refuse("holders must be a contiguous int32 tensor from page_holders(%lld) on cuda:%d, got %s", (long long)num_pages, dev,
           describe(t).c_str());
  return t.data_ptr<int32_t>();
}

// (src, dst, rows, lens, pages, table, holders, page_size, status, refused) -> (lens, pages)
PyObject* fork(PyObject* const* a) {
  const at::Tensor& lens = tensor(a[3], "lens");
  const int dev = cuda_index(lens);
  const int64_t n = lens.numel();
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  int64_t m;
  const int32_t* src = i32(a[0], "src", -1, dev, &m);
  const int32_t *dst = i32(a[1], "dst", m, dev), *rows = i32_or_none(a[2], "rows", m, dev), *l = i32(a[3], "lens", n, dev),
                *p = i32(a[4], "pages", n, dev);
  const Table t = table_of(a[5], n, dev);
  int32_t* h = holders_of(a[6], -1, dev);
  const int page_size = int32(a[7], "page_size");
  int32_t *s = status_of(a[8], dev), *refused = i32_or_none(a[9], "refused", n, dev);
  if (m > DFLASH_PAGED_MAX_SEQS) refuse("%lld forks, at most %d", (long long)m, DFLASH_PAGED_MAX_SEQS);
  const at::Tensor out = empty({2 * n}, at::kInt, dev);
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_fork", lib.fork, dev, src, dst, rows, (int)m, l, p, (int)n, page_size, t.data, t.ld, t.width, h,
       (int)tensor(a[6], "holders").size(1), o, o + n, refused, s);
  return tuple(slice(out, 0, n), slice(out, n, n));
}

// (lens, new_rows, pages, table, free_pages, head, holders, page_size, num_slots, status, refused)
//   -> (starts, slots, lens, pages, head, copies)
PyObject* reserve_forked(PyObject* const* a) {
  const at::Tensor& lens = tensor(a[0], "lens");
  const int dev = cuda_index(lens);
  const int64_t n = lens.numel(), num_slots = int32(a[8], "num_slots");
  const int page_size = int32(a[7], "page_size");
  if (num_slots < 0) refuse("num_slots %lld", (long long)num_slots);
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[3], n, dev);
  int64_t num_pages;
  int32_t *l = i32(a[0], "lens", n, dev), *r = i32(a[1], "new_rows", n, dev), *p = i32(a[2], "pages", n, dev),
          *f = i32(a[4], "free_pages", -1, dev, &num_pages), *h = i32(a[5], "head", 1, dev),
          *shared = holders_of(a[6], num_pages, dev), *s = status_of(a[9], dev), *refused = i32_or_none(a[10], "refused", n, dev);
  const at::Tensor out = empty({6 * n + 2 + num_slots}, at::kInt, dev);   // [starts | lens | pages | head | copies | slots]
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_reserve_forked", lib.reserve_forked, dev, l, r, p, (int)n, page_size, t.data, t.ld, t.width, f,
       (int)num_pages, h, shared, o, o + 6 * n + 2, (int)num_slots, o + n + 1, o + 2 * n + 1, o + 3 * n + 1, o + 3 * n + 2, refused,
       s);
  PyObject* copies = THPVariable_Wrap(out.narrow(0, 3 * n + 2, 3 * n).view({n, 3}));
  if (!copies) throw PyError();
  return tuple(slice(out, 0, n + 1), slice(out, 6 * n + 2, num_slots), slice(out, n + 1, n), slice(out, 2 * n + 1, n),
               slice(out, 3 * n + 1, 1), copies);
}

// (keep, pages, table, free_pages, head, holders, page_size, status)
PyObject* release_forked(PyObject* const* a) {
  const at::Tensor& keep = tensor(a[0], "keep");
  const int dev = cuda_index(keep);
  const int64_t n = keep.numel();
  const int page_size = int32(a[6], "page_size");
  if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
  const Table t = table_of(a[2], n, dev);
  int64_t num_pages;
  int32_t *k = i32(a[0], "keep", n, dev), *p = i32(a[1], "pages", n, dev),
          *f = i32(a[3], "free_pages", -1, dev, &num_pages), *h = i32(a[4], "head", 1, dev),
          *shared = holders_of(a[5], num_pages, dev), *s = status_of(a[7], dev);
  const at::Tensor out = empty({n + 1}, at::kInt, dev);
  int32_t* o = out.data_ptr<int32_t>();
  call("dflash_paged_release_forked", lib.release_forked, dev, k, p, (int)n, page_size, t.data, t.ld, t.width, f, (int)num_pages,
       h, shared, o, o + n, s);
  return tuple(slice(out, 0, n), slice(out, n, 1));
}

// (pools: a list of tensors, copies)
PyObject* copy_pages(PyObject* const* a) {
  if (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) refuse("pools must be a list of tensors from q4_pool()");
  const Py_ssize_t layers = PySequence_Fast_GET_SIZE(a[0]);
  if (layers > INT32_MAX) refuse("too many pools");
  std::vector<uint8_t*> data;
  Pool first{};
  for (Py_ssize_t i = 0; i < layers; ++i) {
    const Pool p = pool_of(PySequence_Fast_GET_ITEM(a[0], i));
    if (i == 0) first = p;
    if (p.pages != first.pages || p.nkv != first.nkv || p.page_size != first.page_size || p.dev != first.dev)
      refuse("pools must have the same shape and device");
    data.push_back(p.data);
  }
  if (layers == 0) Py_RETURN_NONE;
  const at::Tensor& t = tensor(a[1], "copies");
  if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != first.dev || t.dim() != 2 || t.size(1) != 3 ||
      t.size(0) > INT32_MAX || !t.is_contiguous())
    refuse("copies must be a contiguous int32 [n, 3] on cuda:%d, got %s", first.dev, describe(t).c_str());
  call("dflash_q4_copy_pages", lib.copy_pages, first.dev, data.data(), (int)layers, first.pages, first.nkv, first.page_size,
       t.data_ptr<int32_t>(), (int)t.size(0));
  Py_RETURN_NONE;
}

// ---- decode operators
int elem_type(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kHalf: return DFLASH_F16;
    case at::kBFloat16: return DFLASH_BF16;
    case at::kFloat: return DFLASH_F32;
    default: refuse("%s must be f16, bf16 or f32, got %s", name, describe(t).c_str());
  }
}
int device_of(const at::Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse("%s must be on a CUDA device, got %s", name, describe(t).c_str());
  return t.get_device();
}
const at::Tensor& on_device(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef size, int dev) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != dev || !t.sizes().equals(size))
    refuse("%s must be %s %s on cuda:%d, got %s", name, c10::toString(type), (std::ostringstream() << size).str().c_str(), dev,
           describe(t).c_str());
  return t;
}
template <class T>
T* dense(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef size, int dev) {
  const at::Tensor& t = on_device(o, name, type, size, dev);
  if (!t.is_contiguous()) refuse("%s must be contiguous", name);
  return static_cast<T*>(t.data_ptr());
}

// (x, turns, factor, rotary_dim, interleaved, inverse, positions, starts, lens, out) -> out
PyObject* rope(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x");
  const int dev = device_of(x, "x"), type = elem_type(x, "x");
  if (x.dim() != 3) refuse("x must be [rows, heads, dim], got %s", describe(x).c_str());
  const int64_t rows = x.size(0), heads = x.size(1), dim = x.size(2), rot = int32(a[3], "rotary_dim");
  if (rows > INT32_MAX || heads > INT32_MAX || dim > INT32_MAX) refuse("x is too large: %s", describe(x).c_str());
  const double factor = PyFloat_AsDouble(a[2]);
  if (factor == -1.0 && PyErr_Occurred()) throw PyError();
  const double* turns = dense<double>(a[1], "turns", at::kDouble, {rot / 2}, dev);
  const void* positions = nullptr;
  bool wide = false;
  const int32_t *starts = nullptr, *lens = nullptr;
  int64_t n = 0;
  if (a[6] != Py_None) {
    const at::Tensor& t = tensor(a[6], "positions");
    wide = t.scalar_type() == at::kLong;
    positions = wide ? dense<void>(a[6], "positions", at::kLong, {rows}, dev) : dense<void>(a[6], "positions", at::kInt, {rows}, dev);
    if (!positions) positions = turns;   // (no rows)
  } else {
    lens = i32(a[8], "lens", -1, dev, &n);
    if (n > DFLASH_PAGED_MAX_SEQS) refuse("%lld requests, at most %d", (long long)n, DFLASH_PAGED_MAX_SEQS);
    starts = i32(a[7], "starts", n + 1, dev);
  }
  // channels that do not lie side by side are copied first
  const at::Tensor src = x.stride(2) == 1 ? x : x.clone(at::MemoryFormat::Contiguous);
  at::Tensor out;
  if (a[9] == Py_None) {
    out = empty(x.sizes(), x.scalar_type(), dev);
  } else {
    out = on_device(a[9], "out", x.scalar_type(), x.sizes(), dev);
    if (out.stride(2) != 1) refuse("out's channels must lie side by side");
  }
  // (the stride of a single row or head may be anything)
  auto stride = [](const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  call("dflash_rope", lib.rope, dev, src.data_ptr(), stride(src, 0), stride(src, 1), type, (int)rows, (int)heads, (int)dim,
       (int)rot, (int)boolean(a[4]), (int)boolean(a[5]), turns, (float)factor, positions, (int)wide, starts, lens, (int)n,
       out.data_ptr(), stride(out, 0), stride(out, 1));
  return a[9] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[9]);
}

// (logits, drafts, uniforms, temperature: a number or a tensor, probs, counts) -> (accepted, tokens)
PyObject* verify(PyObject* const* a) {
  at::Tensor logits = tensor(a[0], "logits");
  const int dev = device_of(logits, "logits"), type = elem_type(logits, "logits");
  if (logits.dim() != 3 || logits.size(0) > INT32_MAX || logits.size(1) > INT32_MAX || logits.size(2) > INT32_MAX)
    refuse("logits must be [requests, block, vocabulary], got %s", describe(logits).c_str());
  const int64_t n = logits.size(0), block = logits.size(1), vocab = logits.size(2);
  if (block < 1 || vocab < 1) refuse("logits must have rows and entries, got %s", describe(logits).c_str());
  if (logits.stride(2) != 1 && vocab > 1) logits = logits.clone(at::MemoryFormat::Contiguous);
  const int32_t* drafts = dense<int32_t>(a[1], "drafts", at::kInt, {n, block - 1}, dev);
  const float* u = dense<float>(a[2], "uniforms", at::kFloat, {n, block}, dev);
  const float* temps = nullptr;
  double temp = 0.0;
  if (THPVariable_Check(a[3])) {
    temps = dense<float>(a[3], "temperature", at::kFloat, {n}, dev);
  } else {
    temp = PyFloat_AsDouble(a[3]);
    if (temp == -1.0 && PyErr_Occurred()) throw PyError();
  }
  at::Tensor probs;
  if (a[4] != Py_None) {
    probs = on_device(a[4], "draft_probs", at::kFloat, {n, block - 1, vocab}, dev);
    if (probs.stride(2) != 1 && vocab > 1) probs = probs.clone(at::MemoryFormat::Contiguous);
  }
  const int32_t* counts = a[5] == Py_None ? nullptr : dense<int32_t>(a[5], "num_drafts", at::kInt, {n}, dev);
  const at::Tensor out = empty({2 * n}, at::kInt, dev);
  int32_t* o = out.data_ptr<int32_t>();
  const bool sampled = probs.defined() && block > 1;
  call("dflash_verify_drafts", lib.verify, dev, logits.data_ptr(), logits.stride(0), logits.stride(1), type, (int)n, (int)block,
       (int)vocab, drafts, u, temps, (float)temp, sampled ? probs.data_ptr<float>() : nullptr, sampled ? probs.stride(0) : 0,
       sampled ? probs.stride(1) : 0, counts, o, o + n);
  return tuple(slice(out, 0, n), slice(out, n, n));
}

// addresses of the library's entries, in the order of Lib
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int COUNT = sizeof(Lib) / sizeof(void*);
  void* at[COUNT];
  if (n != COUNT) {
    PyErr_Format(PyExc_TypeError, "bind: %d addresses expected", COUNT);
    return nullptr;
  }
  for (int i = 0; i < COUNT; ++i)
    if (!(at[i] = PyLong_AsVoidPtr(a[i]))) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: NULL");
      return nullptr;
    }
  static_assert(std::is_trivially_copyable<Lib>::value, "Lib holds addresses only");
  memcpy(&lib, at, sizeof lib);
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
    method<fork, 10>("fork"),
    method<reserve_forked, 11>("reserve_forked"),
    method<release_forked, 8>("release_forked"),
    method<copy_pages, 2>("copy_pages"),
    method<prefix_plan, 8>("prefix_plan"),
    method<prefix_attention, 16>("prefix_attention"),
    method<rope, 10>("rope"),
    method<verify, 6>("verify"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "dflash_paged", "Paged 4-bit cache operators (see paged.py).", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dflash_paged() { return PyModule_Create(&module); }
