// The common form of the Python entry points in native code: argument checks, output and workspace
// allocation and the library call, for calls whose operands are used as they are (plain CUDA tensors,
// no copy to make, no option beyond those listed at each function). Anything else -- a wrong type,
// shape, dtype, device, stride or alignment, a tensor subclass other than a parameter, an empty batch --
// returns None, and the Python function goes on with its own checks, which copy or raise.
//
// Why: a call of this package is a few microseconds of GPU time at small sizes, and the Python
// wrappers took 10 to 17 us of checks and argument conversion each, so that small calls were bound by
// the host. Time per call, and a decode layer (two calls) of one sequence of 512 tokens: layer
// 32.5 -> 15.6 us, decode of two sequences of 60 tokens 12.6 -> 6.6 (with the append fused
// 16.9 -> 6.7), append of 32 tokens 9.8 -> 4.3, QK-norm + RoPE + append of 32 tokens 15.0 -> 5.3.
//
// The functions take the library's entry points by address (bind), so the module links to nothing but
// torch. Each returns None (not this form), a nonzero int (the library's return code; the caller turns
// it into an exception) or its result.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>

#include "../../include/tileinfer_amd.h"

namespace {

decltype(&ti_kv_append) p_append = nullptr;
decltype(&ti_gqa_decode_plan) p_plan = nullptr;
decltype(&ti_gqa_decode_paged) p_decode = nullptr;
decltype(&ti_gqa_decode_paged_gated) p_decode_gated = nullptr;
decltype(&ti_gqa_decode_paged_append) p_decode_append = nullptr;
decltype(&ti_gqa_prefill_paged) p_prefill = nullptr;
decltype(&ti_gqa_prefill_paged_gated) p_prefill_gated = nullptr;
decltype(&ti_gqa_prefill_workspace_bytes) p_prefill_ws = nullptr;
decltype(&ti_qknorm_rope_append) p_qknorm_append = nullptr;
decltype(&ti_latent_rope_append) p_latent_append = nullptr;
decltype(&ti_latent_decode_workspace_bytes) p_latent_ws = nullptr;
decltype(&ti_latent_decode_paged) p_latent_decode = nullptr;
decltype(&ti_cache_mass_workspace_bytes) p_mass_ws = nullptr;
decltype(&ti_cache_mass) p_mass = nullptr;
decltype(&ti_evict_kvcache) p_evict = nullptr;

// A plain tensor with memory of its own on a GPU, or nullptr.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || !t.has_storage() || t.layout() != at::kStrided || t.is_neg()) {
    return nullptr;
  }
  return &t;
}

uintptr_t address(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); }

int dtype_code(const at::Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return TI_DTYPE_BF16;
  if (t.scalar_type() == at::kHalf) return TI_DTYPE_F16;
  return -1;
}

// Unit element stride, the other strides and the address multiples of `elems` 16-bit elements.
bool aligned_rows(const at::Tensor& t, int64_t elems) {
  const auto st = t.strides();
  const size_t n = st.size();
  if (n == 0 || st[n - 1] != 1 || address(t) % (2 * elems) != 0) return false;
  for (size_t i = 0; i + 1 < n; ++i) {
    if (st[i] % elems != 0) return false;
  }
  return true;
}

bool int32_vector(const at::Tensor& t, int64_t n, const at::Device& dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous() &&
         t.device() == dev;
}

bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

// The operands that decode and prefill share: queries [rows, H_q, D] and one layer's cache pages.
struct Paged {
  const at::Tensor *q, *k, *v, *table;
  int64_t rows_q, hq, hkv, d, rows, page, width, batch;
  int dtype;
};

bool paged(PyObject* const* a, PyObject* page, Paged& o) {
  o.q = plain(a[0]);
  o.k = plain(a[1]);
  o.v = plain(a[2]);
  o.table = plain(a[3]);
  if (!o.q || !o.k || !o.v || !o.table || !PyLong_CheckExact(page)) return false;
  o.page = PyLong_AsLongLong(page);
  if (o.page == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  const at::Tensor &q = *o.q, &k = *o.k, &v = *o.v, &t = *o.table;
  if (q.dim() != 3 || k.dim() != 4 || t.dim() != 2 || k.sizes() != v.sizes()) return false;
  o.rows_q = q.size(0);
  o.hq = q.size(1);
  o.d = q.size(2);
  o.hkv = k.size(2);
  o.rows = k.size(0) * k.size(1);
  o.batch = t.size(0);
  o.width = t.size(1);
  o.dtype = dtype_code(q);
  const at::Device dev = q.device();
  return o.rows_q > 0 && o.batch > 0 && o.width > 0 && o.hkv > 0 && o.hq % o.hkv == 0 &&
         k.size(3) == o.d && o.dtype >= 0 && k.scalar_type() == q.scalar_type() &&
         v.scalar_type() == q.scalar_type() && k.is_contiguous() && v.is_contiguous() &&
         t.scalar_type() == at::kInt && t.stride(1) == 1 && k.device() == dev && v.device() == dev &&
         t.device() == dev && o.page > 0 && o.rows % o.page == 0 && aligned_rows(q, 8) &&
         fits32(o.rows_q) && fits32(o.hq) && fits32(o.d) && fits32(o.page) && fits32(o.width) &&
         fits32(o.batch);
}

// The output gate as contiguous [rows, H_q, D] rows; false where it needs a copy or is wrong.
bool gate_rows(PyObject* o, const Paged& p, const at::Tensor** out) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* g = plain(o);
  if (!g || g->numel() != p.rows_q * p.hq * p.d || g->scalar_type() != p.q->scalar_type() ||
      g->device() != p.q->device() || !g->is_contiguous() || address(*g) % 16 != 0) {
    return false;
  }
  *out = g;
  return true;
}

at::Tensor bytes_on(const at::Tensor& like, int64_t n) {
  return at::empty({n}, like.options().dtype(at::kByte));
}

void* stream_of(PyObject* o) { return PyLong_AsVoidPtr(o); }

// Lets other Python threads run while the library call and the allocations before it do (an
// allocation may wait for the GPU, a launch for room in its queue). Restored on every way out.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

PyObject* guarded(PyObject* (*f)(PyObject* const*), PyObject* const* a, Py_ssize_t n, Py_ssize_t want) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return nullptr;
  }
  try {
    return f(a);
  } catch (...) {  // as torch's own functions raise it (out of memory among them)
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

// (q, k_cache, v_cache, block_table, seqlen, page_size, gate | None, key | None, value, slots, stream)
PyObject* decode(PyObject* const* a) {
  Paged p;
  const at::Tensor *gate, *seqlen = plain(a[4]);
  if (!seqlen || !paged(a, a[5], p) || !gate_rows(a[6], p, &gate)) Py_RETURN_NONE;
  const at::Device dev = p.q->device();
  if (p.rows_q != p.batch || !int32_vector(*seqlen, p.batch, dev)) Py_RETURN_NONE;
  const at::Tensor *key = nullptr, *value = nullptr, *slots = nullptr;
  const int64_t row = p.hkv * p.d;
  if (a[7] != Py_None) {
    key = plain(a[7]);
    value = plain(a[8]);
    slots = plain(a[9]);
    if (!key || !value || !slots || gate || !int32_vector(*slots, p.batch, dev)) Py_RETURN_NONE;
    for (const at::Tensor* t : {key, value}) {
      if (t->dim() != 3 || t->size(0) != p.batch || t->size(1) != p.hkv || t->size(2) != p.d ||
          t->scalar_type() != p.q->scalar_type() || t->device() != dev || t->stride(2) != 1 ||
          t->stride(1) != p.d || t->stride(0) < row || !aligned_rows(*t, 8)) {
        Py_RETURN_NONE;
      }
    }
  }
  void* stream = stream_of(a[10]);
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    int32_t split = 0, splits = 0;
    int64_t ws_bytes = 0;
    rc = p_plan(int32_t(p.batch), int32_t(p.hq), int32_t(p.hkv), int32_t(p.d), int32_t(p.page),
                int32_t(p.width), 0, &split, &splits, &ws_bytes);
    if (rc == TI_OK) {
      out = at::empty({p.batch, p.hq, p.d}, p.q->options());
      at::Tensor ws;
      if (ws_bytes > 0) ws = bytes_on(*p.q, ws_bytes);
      void* wp = ws_bytes > 0 ? ws.data_ptr() : nullptr;
      const int32_t* table = static_cast<const int32_t*>(p.table->data_ptr());
      const int32_t* lens = static_cast<const int32_t*>(seqlen->data_ptr());
#define TI_DECODE_ARGS                                                                            \
  p.q->data_ptr(), p.q->stride(0), p.q->stride(1), p.k->data_ptr(), p.v->data_ptr(), table,       \
      p.table->stride(0), lens, out.data_ptr(), wp, ws_bytes, int32_t(p.batch), int32_t(p.hq),    \
      int32_t(p.hkv), int32_t(p.d), int32_t(p.page), p.rows / p.page, int32_t(p.width), 0,        \
      TI_DECODE_AUTO, p.dtype
      if (key) {
        rc = p_decode_append(TI_DECODE_ARGS, key->data_ptr(), value->data_ptr(), key->stride(0),
                             value->stride(0), static_cast<const int32_t*>(slots->data_ptr()),
                             p.rows, stream);
      } else if (gate) {
        rc = p_decode_gated(TI_DECODE_ARGS, gate->data_ptr(), p.hq * p.d, p.d, stream);
      } else {
        rc = p_decode(TI_DECODE_ARGS, stream);
      }
#undef TI_DECODE_ARGS
    }
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
}

// (q, k_cache, v_cache, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q, page_size, causal,
//  per_unit, gate | None, stream)
PyObject* prefill(PyObject* const* a) {
  Paged p;
  const at::Tensor *gate, *cu = plain(a[4]), *lens = plain(a[5]);
  if (!cu || !lens || !PyLong_CheckExact(a[6]) || !paged(a, a[7], p) || !gate_rows(a[10], p, &gate)) {
    Py_RETURN_NONE;
  }
  const at::Device dev = p.q->device();
  const int64_t max_q = PyLong_AsLongLong(a[6]);
  if (max_q == -1 && PyErr_Occurred()) PyErr_Clear();
  if (!fits32(max_q) || !int32_vector(*cu, p.batch + 1, dev) || !int32_vector(*lens, p.batch, dev)) {
    Py_RETURN_NONE;
  }
  const bool causal = a[8] == Py_True, per_unit = a[9] == Py_True;
  void* stream = stream_of(a[11]);
  at::Tensor out;
  int rc = TI_OK;
  {
    Unlocked unlocked;
    int64_t ws_bytes = 0;
    if (!per_unit) {
      rc = p_prefill_ws(int32_t(p.batch), int32_t(p.rows_q), int32_t(p.hq), int32_t(p.hkv),
                        int32_t(p.d), int32_t(p.page), int32_t(p.width), &ws_bytes);
    }
    if (rc == TI_OK) {
      out = at::empty({p.rows_q, p.hq, p.d}, p.q->options());
      at::Tensor ws;
      if (ws_bytes > 0) ws = bytes_on(*p.q, ws_bytes);
      void* wp = ws_bytes > 0 ? ws.data_ptr() : nullptr;
#define TI_PREFILL_ARGS                                                                           \
  p.q->data_ptr(), p.q->stride(0), p.q->stride(1), p.k->data_ptr(), p.v->data_ptr(),              \
      static_cast<const int32_t*>(p.table->data_ptr()), p.table->stride(0),                       \
      static_cast<const int32_t*>(cu->data_ptr()), static_cast<const int32_t*>(lens->data_ptr()), \
      out.data_ptr(), out.stride(0), out.stride(1), wp, ws_bytes, int32_t(p.batch),               \
      int32_t(p.rows_q), int32_t(max_q), int32_t(p.hq), int32_t(p.hkv), int32_t(p.d),             \
      int32_t(p.page), p.rows / p.page, int32_t(p.width), causal ? 1 : 0, p.dtype
      rc = gate ? p_prefill_gated(TI_PREFILL_ARGS, gate->data_ptr(), p.hq * p.d, p.d, stream)
                : p_prefill(TI_PREFILL_ARGS, stream);
#undef TI_PREFILL_ARGS
    }
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
}

// One layer's cache as token rows [num_slots, row], the same strides for K and V.
bool cache_rows(const at::Tensor* k, const at::Tensor* v, int64_t row, const at::Tensor& like) {
  return k->dim() == 2 && k->size(1) == row && k->stride(1) == 1 && k->sizes() == v->sizes() &&
         k->strides() == v->strides() && k->scalar_type() == like.scalar_type() &&
         v->scalar_type() == like.scalar_type() && k->device() == like.device() &&
         v->device() == like.device();
}

// (key, value, k_cache, v_cache, slot_mapping, stream) -> True
PyObject* append(PyObject* const* a) {
  const at::Tensor *key = plain(a[0]), *value = plain(a[1]), *k = plain(a[2]), *v = plain(a[3]),
                   *slots = plain(a[4]);
  if (!key || !value || !k || !v || !slots || key->dim() != 3 || key->sizes() != value->sizes()) {
    Py_RETURN_NONE;
  }
  const int64_t n = key->size(0), h = key->size(1), d = key->size(2);
  const int code = dtype_code(*key);
  if (n <= 0 || h <= 0 || d <= 0 || code < 0 || value->scalar_type() != key->scalar_type() ||
      value->device() != key->device() || !cache_rows(k, v, h * d, *key) ||
      !int32_vector(*slots, n, key->device())) {
    Py_RETURN_NONE;
  }
  for (const at::Tensor* t : {key, value}) {
    if (t->stride(2) != 1 || t->stride(1) != d || t->stride(0) < h * d) Py_RETURN_NONE;
  }
  void* stream = stream_of(a[5]);
  int rc;
  {
    Unlocked unlocked;
    rc = p_append(key->data_ptr(), value->data_ptr(), key->stride(0), value->stride(0),
                  k->data_ptr(), v->data_ptr(), k->stride(0),
                  static_cast<const int32_t*>(slots->data_ptr()), n, h * d, k->size(0), code, stream);
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  Py_RETURN_TRUE;
}

// (q, k, v, q_weight, k_weight, cos, sin, k_cache, v_cache, slot_mapping, eps, stream)
PyObject* qknorm_append(PyObject* const* a) {
  const at::Tensor* t[10];
  for (int i = 0; i < 10; ++i) {
    t[i] = plain(a[i]);
    if (!t[i]) Py_RETURN_NONE;
  }
  const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &qw = *t[3], &kw = *t[4], &cos = *t[5],
                   &sin = *t[6], &slots = *t[9];
  if (!PyFloat_CheckExact(a[10]) || q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes()) {
    Py_RETURN_NONE;
  }
  const int64_t n = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(1);
  const int code = dtype_code(q);
  if (code < 0 || n <= 0 || hq <= 0 || hkv <= 0 || k.size(0) != n || k.size(2) != d ||
      cos.dim() != 2 || cos.size(0) != n || cos.sizes() != sin.sizes() ||
      cos.strides() != sin.strides() || cos.stride(1) != 1) {
    Py_RETURN_NONE;
  }
  const int64_t rd = cos.size(1);
  for (int i = 0; i < 7; ++i) {
    if (t[i]->scalar_type() != q.scalar_type() || t[i]->device() != q.device()) Py_RETURN_NONE;
  }
  for (const at::Tensor* x : {&q, &k, &v}) {
    if (!aligned_rows(*x, 2)) Py_RETURN_NONE;
  }
  for (const at::Tensor* x : {&qw, &kw}) {
    if (x->dim() != 1 || x->size(0) != d || x->stride(0) != 1) Py_RETURN_NONE;
  }
  if (rd > d || rd % 2 || rd == 0 || !fits32(n) || !fits32(hq) || !fits32(hkv) || !fits32(d) ||
      !cache_rows(t[7], t[8], hkv * d, q) || !int32_vector(slots, n, q.device())) {
    Py_RETURN_NONE;
  }
  const float eps = float(PyFloat_AS_DOUBLE(a[10]));
  void* stream = stream_of(a[11]);
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    out = at::empty({n, hq, d}, q.options());
    rc = p_qknorm_append(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
        v.stride(0), v.stride(1), qw.data_ptr(), kw.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        n == 1 ? 0 : cos.stride(0), out.data_ptr(), out.stride(0), out.stride(1), t[7]->data_ptr(),
        t[8]->data_ptr(), t[7]->stride(0), static_cast<const int32_t*>(slots.data_ptr()),
        t[7]->size(0), int32_t(n), int32_t(hq), int32_t(hkv), int32_t(d), int32_t(rd), eps, code,
        stream);
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
}

constexpr int64_t kRope = 64;

bool latent_dim(int64_t n) { return n == 256 || n == 512; }

// A positive, finite float.
bool scale_of(PyObject* o, float& out) {
  if (!PyFloat_CheckExact(o)) return false;
  const double x = PyFloat_AS_DOUBLE(o);
  out = float(x);
  return x > 0 && x < 1e30;
}

bool int_of(PyObject* o, int64_t& out) {
  if (!PyLong_CheckExact(o)) return false;
  out = PyLong_AsLongLong(o);
  if (out == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return fits32(out);
}

// A layer's cache pages, its block table, lengths and page size.
struct Pages {
  const at::Tensor *cache, *table, *lens;
  int64_t rows, page, width, batch;
};

bool pages(PyObject* cache, PyObject* table, PyObject* lens, PyObject* page, Pages& o) {
  o.cache = plain(cache);
  o.table = plain(table);
  o.lens = plain(lens);
  if (!o.cache || !o.table || !o.lens || !int_of(page, o.page) || o.cache->dim() != 4 || o.table->dim() != 2) return false;
  const at::Device dev = o.cache->device();
  o.rows = o.cache->size(0) * o.cache->size(1);
  o.batch = o.table->size(0);
  o.width = o.table->size(1);
  return o.page > 0 && o.rows % o.page == 0 && o.batch > 0 && o.width > 0 && fits32(o.batch) && fits32(o.width) &&
         o.cache->is_contiguous() && address(*o.cache) % 16 == 0 && dtype_code(*o.cache) >= 0 &&
         o.table->scalar_type() == at::kInt && o.table->stride(1) == 1 && o.table->device() == dev &&
         int32_vector(*o.lens, o.batch, dev);
}

// Queries [B, H, D] or [B, N, H, D] of a cache with D values a row.
struct Queries {
  const at::Tensor* q;
  int64_t batch, tokens, heads, dim, st_b, st_t, st_h;
};

bool queries(PyObject* o, const Pages& p, Queries& out) {
  out.q = plain(o);
  if (!out.q) return false;
  const at::Tensor& q = *out.q;
  const int64_t n = q.dim();
  if ((n != 3 && n != 4) || !aligned_rows(q, 8) || q.scalar_type() != p.cache->scalar_type() ||
      q.device() != p.cache->device()) {
    return false;
  }
  out.batch = q.size(0);
  out.tokens = n == 4 ? q.size(1) : 1;
  out.heads = q.size(n - 2);
  out.dim = q.size(n - 1);
  out.st_b = q.stride(0);
  out.st_t = n == 4 ? q.stride(1) : 0;
  out.st_h = q.stride(n - 2);
  return out.batch == p.batch && out.tokens > 0 && out.heads > 0 && out.dim == p.cache->size(3) &&
         fits32(out.tokens) && fits32(out.heads) && fits32(out.dim);
}

// (q_rope | None, latent, key_rope, weight, cos, sin, latent_cache, slot_mapping, eps, weight_offset, stream)
// -> q_out, or True without queries
PyObject* latent_append(PyObject* const* a) {
  const at::Tensor* t[7];  // latent, key_rope, weight, cos, sin, latent_cache, slots
  for (int i = 0; i < 7; ++i) {
    t[i] = plain(a[i + 1]);
    if (!t[i]) Py_RETURN_NONE;
  }
  const at::Tensor &c = *t[0], &k = *t[1], &w = *t[2], &cos = *t[3], &sin = *t[4], &cache = *t[5], &slots = *t[6];
  const int code = dtype_code(c);
  if (!PyFloat_CheckExact(a[8]) || !PyFloat_CheckExact(a[9]) || code < 0 || c.dim() != 2 || k.dim() != 2 ||
      w.dim() != 1 || cos.dim() != 2 || cache.dim() != 2) {
    Py_RETURN_NONE;
  }
  const int64_t n = c.size(0), dim = c.size(1);
  for (int i = 0; i < 6; ++i) {
    if (t[i]->scalar_type() != c.scalar_type() || t[i]->device() != c.device() || !aligned_rows(*t[i], 8)) {
      Py_RETURN_NONE;
    }
  }
  if (n <= 0 || !latent_dim(dim) || k.size(0) != n || k.size(1) != kRope || w.size(0) != dim || cos.size(0) != n ||
      cos.size(1) != kRope || cos.sizes() != sin.sizes() || cos.strides() != sin.strides() ||
      cache.size(1) != dim + kRope || cache.stride(0) < dim + kRope || !int32_vector(slots, n, c.device())) {
    Py_RETURN_NONE;
  }
  const at::Tensor* q = nullptr;
  int64_t heads = 0;
  if (a[0] != Py_None) {
    q = plain(a[0]);
    if (!q || q->dim() != 3 || q->size(0) != n || q->size(1) <= 0 || q->size(2) != kRope ||
        q->scalar_type() != c.scalar_type() || q->device() != c.device() || !aligned_rows(*q, 8)) {
      Py_RETURN_NONE;
    }
    heads = q->size(1);
  }
  if (!fits32(n) || !fits32(heads)) Py_RETURN_NONE;
  void* stream = stream_of(a[10]);
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    if (q) out = at::empty({n, heads, kRope}, q->options());
    rc = p_latent_append(q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0, q ? q->stride(1) : 0,
                         q ? out.data_ptr() : nullptr, heads * kRope, kRope, c.data_ptr(), c.stride(0), k.data_ptr(),
                         k.stride(0), w.data_ptr(), float(PyFloat_AS_DOUBLE(a[9])), cos.data_ptr(), sin.data_ptr(),
                         n == 1 ? 0 : cos.stride(0), cache.data_ptr(), cache.stride(0), cache.size(0),
                         static_cast<const int32_t*>(slots.data_ptr()), int32_t(n), int32_t(heads), int32_t(dim),
                         int32_t(kRope), float(PyFloat_AS_DOUBLE(a[8])), code, stream);
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(out));
}

// (q, latent_cache, block_table, seqlen, page_size, scale, stream)
PyObject* latent_decode(PyObject* const* a) {
  Pages p;
  Queries q;
  float scale;
  if (!pages(a[1], a[2], a[3], a[4], p) || !queries(a[0], p, q) || !scale_of(a[5], scale) || p.cache->size(2) != 1 ||
      !latent_dim(q.dim - kRope)) {
    Py_RETURN_NONE;
  }
  const int64_t dim = q.dim - kRope;
  void* stream = stream_of(a[6]);
  at::Tensor out;
  int rc;
  {
    Unlocked unlocked;
    int64_t ws_bytes = 0;
    rc = p_latent_ws(int32_t(p.batch), int32_t(q.tokens), int32_t(q.heads), int32_t(dim), &ws_bytes);
    if (rc == TI_OK) {
      out = q.q->dim() == 3 ? at::empty({p.batch, q.heads, dim}, q.q->options())
                            : at::empty({p.batch, q.tokens, q.heads, dim}, q.q->options());
      at::Tensor ws = bytes_on(*q.q, ws_bytes);
      rc = p_latent_decode(q.q->data_ptr(), q.st_b, q.st_t, q.st_h, p.cache->data_ptr(),
                           static_cast<const int32_t*>(p.table->data_ptr()), p.table->stride(0),
                           static_cast<const int32_t*>(p.lens->data_ptr()), out.data_ptr(), ws.data_ptr(), ws_bytes,
                           int32_t(p.batch), int32_t(q.tokens), int32_t(q.heads), int32_t(dim), int32_t(kRope),
                           int32_t(p.page), p.rows / p.page, int32_t(p.width), scale, dtype_code(*q.q), stream);
    }
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
}

// Running sums [batch, heads, >= tokens] of a cache's tokens, rows apart.
bool mass_rows(const at::Tensor& m, int64_t batch, int64_t heads, int64_t tokens, const at::Device& dev) {
  return m.scalar_type() == at::kFloat && m.dim() == 3 && m.size(0) == batch && m.size(1) == heads &&
         m.size(2) >= tokens && m.device() == dev && m.stride(2) == 1 && m.stride(1) >= m.size(2) &&
         (batch == 1 || m.stride(0) >= heads * m.stride(1));
}

// (q, k_cache, block_table, seqlen, page_size, scale, mass | None, stream) -> mass
PyObject* cache_mass(PyObject* const* a) {
  Pages p;
  Queries q;
  float scale;
  if (!pages(a[1], a[2], a[3], a[4], p) || !queries(a[0], p, q) || !scale_of(a[5], scale)) Py_RETURN_NONE;
  const int64_t hkv = p.cache->size(2), tokens = p.width * p.page;
  const bool dim_ok = q.dim == 128 || q.dim == 256 || q.dim == 320 || q.dim == 576;
  if (!dim_ok || hkv <= 0 || q.heads % hkv != 0) Py_RETURN_NONE;
  at::Tensor mass;
  if (a[6] != Py_None) {
    const at::Tensor* m = plain(a[6]);
    if (!m || !mass_rows(*m, p.batch, hkv, tokens, q.q->device())) Py_RETURN_NONE;
    mass = *m;
  }
  void* stream = stream_of(a[7]);
  int rc;
  {
    Unlocked unlocked;
    int64_t ws_bytes = 0;
    rc = p_mass_ws(int32_t(p.batch), int32_t(q.tokens), int32_t(q.heads), int32_t(hkv), int32_t(q.dim),
                   int32_t(p.page), int32_t(p.width), &ws_bytes);
    if (rc == TI_OK) {
      if (!mass.defined()) mass = at::zeros({p.batch, hkv, tokens}, q.q->options().dtype(at::kFloat));
      at::Tensor ws = bytes_on(*q.q, ws_bytes);
      rc = p_mass(q.q->data_ptr(), q.st_b, q.st_t, q.st_h, p.cache->data_ptr(),
                  static_cast<const int32_t*>(p.table->data_ptr()), p.table->stride(0),
                  static_cast<const int32_t*>(p.lens->data_ptr()), static_cast<float*>(mass.data_ptr()),
                  mass.stride(0), mass.stride(1), ws.data_ptr(), ws_bytes, int32_t(p.batch), int32_t(q.tokens),
                  int32_t(q.heads), int32_t(hkv), int32_t(q.dim), int32_t(p.page), p.rows / p.page,
                  int32_t(p.width), scale, dtype_code(*q.q), stream);
    }
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  if (a[6] != Py_None) return (Py_INCREF(a[6]), a[6]);
  return THPVariable_Wrap(std::move(mass));
}

// (k_cache, v_cache | None, mass, block_table, seqlen, new_block_table, budget, page_size, sinks, recent, stream)
// -> (new_seqlen, kept, new_mass)
PyObject* evict(PyObject* const* a) {
  Pages p;
  const at::Tensor *mass = plain(a[2]), *into = plain(a[5]), *v = nullptr;
  int64_t budget, sinks, recent;
  if (!mass || !into || !pages(a[0], a[3], a[4], a[7], p) || !int_of(a[6], budget) || !int_of(a[8], sinks) ||
      !int_of(a[9], recent)) {
    Py_RETURN_NONE;
  }
  const at::Device dev = p.cache->device();
  const int64_t hkv = p.cache->size(2), dim = p.cache->size(3), tokens = p.width * p.page;
  if (hkv <= 0 || dim <= 0 || dim % 8 != 0 || !fits32(hkv) || !fits32(dim) || budget <= 0 || sinks + recent > budget ||
      !mass_rows(*mass, p.batch, hkv, tokens, dev) || into->dim() != 2 || into->size(0) != p.batch ||
      into->scalar_type() != at::kInt || into->stride(1) != 1 || into->device() != dev || !fits32(into->size(1))) {
    Py_RETURN_NONE;
  }
  if (a[1] != Py_None) {
    v = plain(a[1]);
    if (!v || v->sizes() != p.cache->sizes() || v->scalar_type() != p.cache->scalar_type() || v->device() != dev ||
        !v->is_contiguous() || address(*v) % 16 != 0) {
      Py_RETURN_NONE;
    }
  }
  void* stream = stream_of(a[10]);
  at::Tensor lens, kept, sums;
  int rc;
  {
    Unlocked unlocked;
    const auto ints = p.table->options();
    lens = at::empty({p.batch}, ints);
    kept = at::empty({p.batch, hkv, budget}, ints);
    sums = at::empty({p.batch, hkv, mass->size(2)}, mass->options());
    rc = p_evict(p.cache->data_ptr(), v ? v->data_ptr() : nullptr, static_cast<const float*>(mass->data_ptr()),
                 mass->stride(0), mass->stride(1), mass->size(2), static_cast<const int32_t*>(p.table->data_ptr()),
                 p.table->stride(0), static_cast<const int32_t*>(p.lens->data_ptr()),
                 static_cast<const int32_t*>(into->data_ptr()), into->stride(0),
                 static_cast<int32_t*>(kept.data_ptr()), static_cast<int32_t*>(lens.data_ptr()),
                 static_cast<float*>(sums.data_ptr()), int32_t(p.batch), int32_t(hkv), int32_t(dim),
                 int32_t(p.page), p.rows / p.page, int32_t(p.width), int32_t(into->size(1)), int32_t(budget),
                 int32_t(sinks), int32_t(recent), dtype_code(*p.cache), stream);
  }
  if (rc != TI_OK) return PyLong_FromLong(rc);
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(lens)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(kept)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(sums)));
  return r;
}

// The library's entry points by address, in the order of the list below.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void** slots[] = {(void**)&p_append,        (void**)&p_plan,          (void**)&p_decode,
                    (void**)&p_decode_gated,  (void**)&p_decode_append, (void**)&p_prefill,
                    (void**)&p_prefill_gated, (void**)&p_prefill_ws,    (void**)&p_qknorm_append,
                    (void**)&p_latent_append, (void**)&p_latent_ws,     (void**)&p_latent_decode,
                    (void**)&p_mass_ws,       (void**)&p_mass,          (void**)&p_evict};
  if (n != Py_ssize_t(sizeof(slots) / sizeof(slots[0]))) {
    PyErr_SetString(PyExc_TypeError, "bind: one address for each entry point");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    void* f = PyLong_AsVoidPtr(a[i]);
    if (!f) return nullptr;
    *slots[i] = f;
  }
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(F, a, n, N);
}

#define TI_METHOD(name, n) \
  {#name, (PyCFunction)(void (*)(void))entry<name, n>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         TI_METHOD(decode, 11),
                         TI_METHOD(prefill, 12),
                         TI_METHOD(append, 6),
                         TI_METHOD(qknorm_append, 12),
                         TI_METHOD(latent_append, 11),
                         TI_METHOD(latent_decode, 7),
                         TI_METHOD(cache_mass, 8),
                         TI_METHOD(evict, 11),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycalls", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for (given by the build): the versions whose structures this file was compiled against.
PyMODINIT_FUNC PyInit__pycalls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", TI_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
