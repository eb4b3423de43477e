// Python binding of the paged operators of a decode step: argument checks,
// outputs and the call into the C ABI in one native function each.
//
// Such a call is launched once or more per layer and token, and on the GPU it
// takes a few microseconds; the same checks written in Python, with the 44
// arguments of hc_rope_append converted one by one, took 14 us of host time.
// Every check is made on every call: nothing is kept from one call to the
// next.  A function returns its outputs, or the C ABI's status as an int if
// that is not 0; what the arguments get wrong raises ValueError or TypeError
// before anything is allocated or launched.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <initializer_list>
#include <string>

#include "heterocache_b200.h"

namespace {

constexpr int64_t kD = 128, kPage = HC_PAGE_SIZE, kBlocks = HC_PAGE_SIZE / HC_SPARSE_BLOCK;

struct Refusal {
  PyObject* type;
  std::string what;
};
struct PyErrorIsSet {};  // a Python call failed

[[noreturn]] void refuse(const std::string& what) { throw Refusal{PyExc_ValueError, "heterocache_b200: " + what}; }

using at::Tensor;

[[noreturn]] void not_a_tensor(const char* name) {
  throw Refusal{PyExc_TypeError, std::string("heterocache_b200: ") + name + " must be a tensor"};
}
const Tensor* opt_tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) not_a_tensor(name);
  return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o, const char* name) {
  const Tensor* t = opt_tensor(o, name);
  if (!t) not_a_tensor(name);
  return *t;
}
int integer(PyObject* o, const char* name) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw PyErrorIsSet{};
  if (x < INT_MIN || x > INT_MAX) refuse(std::string(name) + " does not fit 32 bits");
  return (int)x;
}
float number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw PyErrorIsSet{};
  return (float)x;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HC_F32;
    case at::kBFloat16: return HC_BF16;
    case at::kHalf: return HC_F16;
    default:
      throw Refusal{PyExc_TypeError, std::string("heterocache_b200: unsupported dtype ") + c10::toString(t)};
  }
}

// A tensor of contiguous 128-element rows.
const Tensor& rows(const Tensor& t, const char* name) {
  const int64_t n = t.dim();
  if (n == 0 || t.size(n - 1) != kD || t.stride(n - 1) != 1)
    refuse(std::string(name) + " must have a contiguous last dim of 128");
  return t;
}
// A tensor of 128-element rows that is written to: no two rows may share
// memory.  (By increasing stride, each dimension steps over all of those before.)
void apart(const Tensor& t, const char* name) {
  int64_t dims[3], n = 0, span = kD;
  for (int64_t d = 0; d < t.dim() - 1; ++d)
    if (t.size(d) > 1) dims[n++] = d;
  std::sort(dims, dims + n, [&](int64_t a, int64_t b) { return t.stride(a) < t.stride(b); });
  for (int64_t i = 0; i < n; ++i) {
    const int64_t s = t.stride(dims[i]);
    if (s < span) refuse(std::string(name) + " must not overlap itself");
    span += s * (t.size(dims[i]) - 1);
  }
}
// A contiguous int32 tensor of at least n entries.
void ints(const Tensor& t, const char* name, int64_t n, const char* what) {
  if (t.scalar_type() != at::kInt || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous int32 tensor");
  if (t.numel() < n) refuse(what);
}
void ints(const Tensor& t, const char* name) { ints(t, name, 0, ""); }

int narrow(int64_t x, const char* what) {
  if (x > INT_MAX) refuse(std::string(what) + " does not fit 32 bits");
  return (int)x;
}

// A page pool; returns its number of pages.
int pool(const Tensor& t, const char* name, at::ScalarType dtype) {
  if (t.dim() != 4 || t.size(1) != kPage || t.size(2) != 1 || t.size(3) != kD || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous [n_blocks, 256, 1, 128] pool");
  if (t.scalar_type() != dtype) refuse(std::string(name) + " must have the dtype of the other operands");
  return narrow(t.size(0), name);
}
int pools(const Tensor& k, const Tensor& v, at::ScalarType dtype) {
  const int n = pool(k, "k_pool", dtype);
  if (pool(v, "v_pool", dtype) != n) refuse("k_pool and v_pool must have the same shape");
  return n;
}
// The page table's and the lengths' rows; returns the table's width.
int cache_rows(const Tensor& table, const Tensor& lens, int64_t n) {
  const char* what = "block_table and heads_len need a row per (batch row, KV head)";
  ints(table, "block_table");
  if (table.dim() != 2 || table.size(0) < n) refuse(what);
  ints(lens, "heads_len", n, what);
  return narrow(table.size(1), "the width of block_table");
}
void check_bounds(const Tensor& t, int64_t n_pages, at::ScalarType dtype) {
  if (t.scalar_type() != dtype || t.dim() != 4 || t.size(0) != n_pages || t.size(1) != kBlocks || t.size(2) != 2 ||
      t.size(3) != kD || !t.is_contiguous())
    refuse("bounds must be a contiguous [n_blocks, 4, 2, 128] tensor in the pool dtype");
}
void check_err(const Tensor& t) { ints(t, "err", 1, "err needs an entry"); }

void same_device(const Tensor& q, std::initializer_list<const Tensor*> ts) {
  const at::Device d = q.device();
  for (const Tensor* t : ts)
    if (t && t->device() != d)
      refuse("tensors on different devices (" + d.str() + " and " + t->device().str() + ")");
  if (!d.is_cuda()) refuse("tensors must live on a CUDA device");
}

template <typename T = void> T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T = void> T* ptr(const Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
int32_t* iptr(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
int32_t* iptr(const Tensor* t) { return t ? static_cast<int32_t*>(t->data_ptr()) : nullptr; }

void* stream_of(const Tensor& q) { return c10::cuda::getCurrentCUDAStream(q.get_device()).stream(); }

PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// The caller's scratch buffer, of at least n bytes (Workspace.get).
at::Tensor scratch(PyObject* workspace, size_t n, const Tensor& q) {
  static PyObject* get = PyUnicode_InternFromString("get");
  PyObject* size = PyLong_FromSize_t(n);
  if (!size) throw PyErrorIsSet{};
  PyObject* buf = PyObject_CallMethodObjArgs(workspace, get, size, nullptr);
  Py_DECREF(size);
  if (!buf) throw PyErrorIsSet{};
  if (!THPVariable_Check(buf)) {
    Py_DECREF(buf);
    throw Refusal{PyExc_TypeError, "heterocache_b200: the workspace must hold a tensor"};
  }
  at::Tensor t = THPVariable_Unpack(buf);
  Py_DECREF(buf);
  if (t.device() != q.device())
    refuse("tensors on different devices (" + q.device().str() + " and " + t.device().str() + ")");
  if (!t.is_contiguous() || t.scalar_type() != at::kByte) refuse("the workspace must hold contiguous bytes");
  return t;
}

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F body) {
  HANDLE_TH_ERRORS
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "heterocache_b200: %zd arguments in place of %zd", got, want);
    return nullptr;
  }
  try {
    return body();
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.what.c_str());
  } catch (const PyErrorIsSet&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

struct Trig {
  int64_t batch, token;
};
// Batch and token stride of cos or sin, [bsz or 1, T, D] or [T, D].
Trig trig_strides(const Tensor& t, const char* name, int64_t bsz, int64_t T, at::ScalarType dtype,
                  at::ScalarType trig) {
  rows(t, name);
  const int64_t n = t.dim();
  if ((n != 3 && n != 2) || t.size(n - 2) != T || (n == 3 && t.size(0) != 1 && t.size(0) != bsz))
    refuse(std::string(name) + " needs [bsz or 1, tokens, D]");
  if (t.scalar_type() != trig || (trig != dtype && trig != at::kFloat))
    refuse("cos and sin must share a dtype: the queries', or float32");
  return {n == 2 || t.size(0) == 1 ? 0 : t.stride(0), t.stride(n - 2)};
}

PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&]() -> PyObject* {
    const Tensor &q = rows(tensor(a[0], "q"), "q"), &k = rows(tensor(a[1], "k"), "k"),
                 &v = rows(tensor(a[2], "v"), "v");
    const Tensor &cos = tensor(a[3], "cos"), &sin = tensor(a[4], "sin");
    const Tensor &kp = tensor(a[5], "k_pool"), &vp = tensor(a[6], "v_pool"), &table = tensor(a[7], "block_table"),
                 &lens = tensor(a[8], "heads_len"), &free_blocks = tensor(a[9], "free_blocks"),
                 &free_ptr = tensor(a[10], "free_ptr"), &err = tensor(a[11], "err"),
                 &counter = tensor(a[12], "counter");
    const Tensor *counts = opt_tensor(a[13], "counts"), *q_out = opt_tensor(a[14], "q_out"),
                 *lens_out = opt_tensor(a[15], "heads_len_out"), *bounds = opt_tensor(a[16], "bounds");
    if (q.dim() != 4 || k.dim() != 4) refuse("q, k, v need [bsz, heads, tokens, D]");
    const int64_t bsz = q.size(0), H = q.size(1), T = q.size(2), KV = k.size(1);
    const at::ScalarType dtype = q.scalar_type(), trig = cos.scalar_type();
    const int dt = dtype_code(dtype);
    if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
      refuse("k and v must have the same shape and dtype");
    if (k.size(0) != bsz || k.size(2) != T || k.scalar_type() != dtype)
      refuse("q, k and v must share batch, tokens and dtype");
    const int64_t R = bsz * KV;
    if (R <= 0 || H <= 0) refuse("q, k and v need at least one sequence and one head");
    const int n_pages = pools(kp, vp, dtype);
    const int width = cache_rows(table, lens, R);
    ints(free_blocks, "free_blocks");
    ints(free_ptr, "free_ptr", 1, "free_ptr and err need an entry");
    ints(err, "err", 1, "free_ptr and err need an entry");
    ints(counter, "counter", 1, "the workspace's counter needs an entry");
    const Trig c = trig_strides(cos, "cos", bsz, T, dtype, trig), s = trig_strides(sin, "sin", bsz, T, dtype, trig);
    if (counts) ints(*counts, "counts", bsz, "counts needs an entry per sequence");
    if (q_out && (rows(*q_out, "q_out").sizes() != q.sizes() || q_out->scalar_type() != dtype))
      refuse("q_out must have the queries' shape and dtype");
    if (q_out && q_out->numel()) apart(*q_out, "q_out");
    if (lens_out) ints(*lens_out, "heads_len_out", R, "heads_len_out needs a row per (batch row, KV head)");
    if (bounds) check_bounds(*bounds, n_pages, dtype);
    same_device(q, {&k, &v, &cos, &sin, &kp, &vp, &table, &lens, lens_out, &free_blocks, &free_ptr, &err, counts, q_out,
                    bounds, &counter});
    c10::cuda::CUDAGuard guard(q.device());
    at::Tensor made;
    if (!q_out) made = at::empty(q.sizes(), q.options());
    const Tensor& out = q_out ? *q_out : made;
    const int rc = hc_rope_append(
        dt, dtype_code(trig), narrow(bsz, "bsz"), narrow(H, "heads"), narrow(KV, "heads"), narrow(T, "tokens"), (int)kD,
        ptr(q), q.stride(0), q.stride(1), q.stride(2), ptr(k), k.stride(0), k.stride(1), k.stride(2), ptr(v),
        v.stride(0), v.stride(1), v.stride(2), ptr(cos), c.batch, c.token, ptr(sin), s.batch, s.token, ptr(out),
        out.stride(0), out.stride(1), out.stride(2), iptr(counts), ptr(kp), ptr(vp), n_pages, iptr(table), width,
        iptr(lens), iptr(lens_out ? *lens_out : lens), iptr(free_blocks), narrow(free_blocks.numel(), "free_blocks"),
        iptr(free_ptr), ptr(bounds), iptr(counter), iptr(err), stream_of(q));
    if (rc) return PyLong_FromLong(rc);
    return q_out ? same(a[14]) : wrap(std::move(made));
  });
}

// A decode step's query [bsz, H, 1, D].
struct Query {
  int bsz, H, KV, G;
  int64_t sb, sh, R;
  at::ScalarType dtype;
};
Query decode_query(const Tensor& q, PyObject* num_kv_heads, const char* name) {
  rows(q, "q");
  const int KV = integer(num_kv_heads, "num_kv_heads");
  if (q.dim() != 4 || q.size(2) != 1) refuse(std::string(name) + " takes one query position, [bsz, H, 1, D]");
  const int64_t bsz = q.size(0), H = q.size(1);
  if (bsz <= 0 || KV <= 0 || H <= 0 || H % KV)
    refuse("the " + std::to_string(H) + " query heads do not split evenly over " + std::to_string(KV) + " KV heads");
  return {narrow(bsz, "bsz"), narrow(H, "heads"), KV, (int)(H / KV), q.stride(0), q.stride(1), bsz * KV,
          q.scalar_type()};
}

void check_out(const Tensor* out, const Tensor& q) {
  if (out && (!out->is_contiguous() || out->numel() != q.numel() || out->scalar_type() != q.scalar_type()))
    refuse("out must be a contiguous [bsz, H, D] buffer in the query dtype");
}
at::Tensor out_or_new(const Tensor* out, const Tensor& q) {
  return out ? *out : at::empty({q.size(0), q.size(1), kD}, q.options());
}

PyObject* flash_decode_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0], "q"), &kp = tensor(a[1], "k_pool"), &vp = tensor(a[2], "v_pool"),
                 &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "heads_len"),
                 &shared = tensor(a[5], "shared_len");
    const Tensor *out = opt_tensor(a[7], "out"), *kn = opt_tensor(a[11], "k_new"), *vn = opt_tensor(a[12], "v_new");
    const Tensor& err = tensor(a[10], "err");
    const float scale = number(a[8]);
    const Query x = decode_query(q, a[6], "decode attention");
    const int n_pages = pools(kp, vp, x.dtype);
    const int width = cache_rows(table, lens, x.R);
    check_out(out, q);
    ints(shared, "shared_len", x.KV, "shared_len needs an entry per KV head");
    check_err(err);
    if (!kn != !vn) refuse("k_new and v_new come together");
    if (kn) {
      rows(*kn, "k_new"), rows(*vn, "v_new");
      if (kn->sizes() != vn->sizes() || kn->scalar_type() != vn->scalar_type())
        refuse("k and v must have the same shape and dtype");
      if (kn->dim() != 4 || kn->size(0) != x.bsz || kn->size(1) != x.KV || kn->size(2) != 1 ||
          kn->scalar_type() != x.dtype)
        refuse("k_new/v_new must be [bsz, KV, 1, D] in the query dtype");
    }
    const int dt = dtype_code(x.dtype);
    same_device(q, {&kp, &vp, &table, &lens, &shared, out, &err, kn, vn});
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor ws =
        scratch(a[9], hc_flash_decode_shared_workspace_size(dt, x.bsz, x.KV, x.G, (int)kD), q);
    at::Tensor o = out_or_new(out, q);
    const int rc = hc_flash_decode_shared(
        dt, x.bsz, x.KV, x.G, (int)kD, ptr(q), x.sb, x.sh, ptr(kp), ptr(vp), n_pages, iptr(table), width, iptr(lens),
        iptr(shared), ptr(kn), ptr(vn), kn ? kn->stride(0) : 0, kn ? kn->stride(1) : 0, kn ? vn->stride(0) : 0,
        kn ? vn->stride(1) : 0, scale, ptr(o), ptr(ws), (size_t)ws.numel(), iptr(err), stream_of(q));
    if (rc) return PyLong_FromLong(rc);
    return out ? same(a[7]) : wrap(std::move(o));
  });
}

PyObject* block_bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Tensor &kp = tensor(a[0], "k_pool"), &table = tensor(a[1], "block_table"), &lens = tensor(a[2], "heads_len"),
                 &bounds = tensor(a[3], "bounds"), &err = tensor(a[4], "err");
    const Tensor* list = opt_tensor(a[5], "rows");
    const int last = integer(a[6], "last");
    const at::ScalarType dtype = kp.scalar_type();
    const int n_pages = pool(kp, "k_pool", dtype);
    const int64_t R = table.dim() ? table.size(0) : 0;
    const int width = cache_rows(table, lens, R);
    check_bounds(bounds, n_pages, dtype);
    check_err(err);
    if (last < 0) refuse("last must not be negative");
    if (list) ints(*list, "rows");
    const int dt = dtype_code(dtype);
    same_device(kp, {&table, &lens, &bounds, &err, list});
    if (list && list->numel() == 0) return same(a[3]);  // no rows (a null pointer would be all of them)
    c10::cuda::CUDAGuard guard(kp.device());
    const int rc = hc_block_bounds(dt, narrow(R, "rows"), (int)kD, ptr(kp), n_pages, iptr(table), width, iptr(lens),
                                   iptr(list), list ? narrow(list->numel(), "rows") : 0, last, ptr(bounds), iptr(err),
                                   stream_of(kp));
    if (rc) return PyLong_FromLong(rc);
    return same(a[3]);
  });
}

// The selection's own operands.
struct Select {
  int n, sink, recent;
  const Tensor *blocks, *counts;
};
Select select_args(PyObject* n_select, PyObject* sink, PyObject* recent, PyObject* blocks, PyObject* counts,
                   int64_t R) {
  Select s = {integer(n_select, "n_select"), integer(sink, "sink"), integer(recent, "recent"),
              opt_tensor(blocks, "blocks"), opt_tensor(counts, "counts")};
  if (s.n < 1 || s.sink < 0 || s.recent < 0 || (int64_t)s.sink + s.recent > s.n)
    refuse("sink + recent blocks must not be more than n_select, which must be at least 1");
  const char* what = "blocks needs [rows, n_select] and counts an entry per row";
  if (s.blocks) {
    ints(*s.blocks, "blocks");
    if (s.blocks->dim() != 2 || s.blocks->size(0) != R || s.blocks->size(1) != s.n) refuse(what);
  }
  if (s.counts) ints(*s.counts, "counts", R, what);
  return s;
}

PyObject* block_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0], "q"), &bounds = tensor(a[1], "bounds"), &table = tensor(a[2], "block_table"),
                 &lens = tensor(a[3], "heads_len"), &err = tensor(a[9], "err");
    const Query x = decode_query(q, a[4], "block_select");
    const int width = cache_rows(table, lens, x.R);
    const int64_t n_pages = bounds.dim() ? bounds.size(0) : 0;
    check_bounds(bounds, n_pages, x.dtype);
    check_err(err);
    const Select s = select_args(a[5], a[6], a[7], a[10], a[11], x.R);
    const int dt = dtype_code(x.dtype);
    same_device(q, {&bounds, &table, &lens, &err, s.blocks, s.counts});
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor ws = scratch(a[8], hc_block_select_workspace_size(x.bsz, x.KV, width), q);
    at::Tensor blocks = s.blocks ? *s.blocks : at::empty({x.R, s.n}, q.options().dtype(at::kInt));
    at::Tensor counts = s.counts ? *s.counts : at::empty({x.R}, q.options().dtype(at::kInt));
    const int rc = hc_block_select(dt, x.bsz, x.KV, x.G, (int)kD, ptr(q), x.sb, x.sh, ptr(bounds),
                                   narrow(n_pages, "bounds"), iptr(table), width, iptr(lens), s.n, s.sink, s.recent,
                                   iptr(blocks), iptr(counts), ptr(ws), (size_t)ws.numel(), iptr(err), stream_of(q));
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("(NN)", s.blocks ? same(a[10]) : wrap(std::move(blocks)),
                         s.counts ? same(a[11]) : wrap(std::move(counts)));
  });
}

PyObject* flash_decode_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0], "q"), &kp = tensor(a[1], "k_pool"), &vp = tensor(a[2], "v_pool"),
                 &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "heads_len"),
                 &blocks = tensor(a[5], "blocks"), &counts = tensor(a[6], "counts"), &err = tensor(a[11], "err");
    const Tensor* out = opt_tensor(a[8], "out");
    const float scale = number(a[9]);
    const Query x = decode_query(q, a[7], "decode attention");
    const int n_pages = pools(kp, vp, x.dtype);
    const int width = cache_rows(table, lens, x.R);
    check_out(out, q);
    const char* what = "blocks needs [rows, n] and counts an entry per row";
    ints(blocks, "blocks", 1, what);
    ints(counts, "counts", x.R, what);
    check_err(err);
    if (blocks.dim() != 2 || blocks.size(0) < x.R) refuse(what);
    const int dt = dtype_code(x.dtype);
    same_device(q, {&kp, &vp, &table, &lens, &blocks, &counts, out, &err});
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor ws = scratch(a[10], hc_flash_decode_workspace_size(x.bsz, x.KV, x.G, (int)kD), q);
    at::Tensor o = out_or_new(out, q);
    const int rc = hc_flash_decode_blocks(dt, x.bsz, x.KV, x.G, (int)kD, ptr(q), x.sb, x.sh, ptr(kp), ptr(vp), n_pages,
                                          iptr(table), width, iptr(lens), iptr(blocks), iptr(counts),
                                          narrow(blocks.size(1), "blocks"), scale, ptr(o), ptr(ws),
                                          (size_t)ws.numel(), iptr(err), stream_of(q));
    if (rc) return PyLong_FromLong(rc);
    return out ? same(a[8]) : wrap(std::move(o));
  });
}

PyObject* flash_decode_sparse(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0], "q"), &kp = tensor(a[1], "k_pool"), &vp = tensor(a[2], "v_pool"),
                 &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "heads_len"),
                 &bounds = tensor(a[5], "bounds"), &err = tensor(a[13], "err");
    const Tensor* out = opt_tensor(a[10], "out");
    const float scale = number(a[11]);
    const Query x = decode_query(q, a[6], "decode attention");
    const int n_pages = pools(kp, vp, x.dtype);
    const int width = cache_rows(table, lens, x.R);
    check_out(out, q);
    check_bounds(bounds, n_pages, x.dtype);
    check_err(err);
    const Select s = select_args(a[7], a[8], a[9], a[14], a[15], x.R);
    const int dt = dtype_code(x.dtype);
    same_device(q, {&kp, &vp, &table, &lens, &bounds, s.blocks, s.counts, out, &err});
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor ws =
        scratch(a[12], hc_flash_decode_sparse_workspace_size(x.bsz, x.KV, x.G, (int)kD, width), q);
    at::Tensor o = out_or_new(out, q);
    at::Tensor blocks = s.blocks ? *s.blocks : at::empty({x.R, s.n}, q.options().dtype(at::kInt));
    at::Tensor counts = s.counts ? *s.counts : at::empty({x.R}, q.options().dtype(at::kInt));
    const int rc = hc_flash_decode_sparse(dt, x.bsz, x.KV, x.G, (int)kD, ptr(q), x.sb, x.sh, ptr(kp), ptr(vp), n_pages,
                                          iptr(table), width, iptr(lens), ptr(bounds), s.n, s.sink, s.recent, scale,
                                          ptr(o), iptr(blocks), iptr(counts), ptr(ws), (size_t)ws.numel(), iptr(err),
                                          stream_of(q));
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("(NNN)", out ? same(a[10]) : wrap(std::move(o)),
                         s.blocks ? same(a[14]) : wrap(std::move(blocks)),
                         s.counts ? same(a[15]) : wrap(std::move(counts)));
  });
}

#define HC_ENTRY(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {HC_ENTRY(rope_append),
                          HC_ENTRY(flash_decode_shared),
                          HC_ENTRY(block_bounds),
                          HC_ENTRY(block_select),
                          HC_ENTRY(flash_decode_blocks),
                          HC_ENTRY(flash_decode_sparse),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged", "Native calls of heterocache_b200.ops.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged() { return PyModule_Create(&kModule); }
