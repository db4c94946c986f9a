// The host side of heads.py: checks a call's tensors, allocates its results and workspace from torch, lays its structs out
// and calls the C ABI.  A decoding step's kernels take a few microseconds each, and the same work in Python (attribute
// lookups, tuples, ctypes objects) took 13 to 18 microseconds a call; here a call takes 5 to 6.5 of host time, its
// results' allocation and the launch included, the backward with five allocations and two launches 11.
//
// The entry points come as addresses from the ctypes binding (bind), so that this module and _lib.py use one library.
// No C++ exception leaves a function: whatever is thrown becomes a Python one.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include "../../include/dfdx_b200.h"
#include <string>

namespace {

struct Entries {
  decltype(&b200_qk_norm_rotary_forward) forward = nullptr;
  decltype(&b200_qk_norm_rotary_backward) backward = nullptr;
  decltype(&b200_qk_norm_rotary_backward_workspace_bytes) backward_bytes = nullptr;
  decltype(&b200_kv_cache_append) append = nullptr;
  decltype(&b200_kv_cache_read) read = nullptr;
  decltype(&b200_kv_cache_attention) attention = nullptr;
  decltype(&b200_kv_cache_attention_workspace_bytes) attention_bytes = nullptr;
} entry;
PyObject *shape_mismatch = nullptr, *check_status = nullptr;       // ShapeMismatch; _lib.check(status, where)

// What a check throws: a Python exception type and its text; or nothing but the fact that one is set already.
struct Refused {
  PyObject* type;
  std::string text;
};
[[noreturn]] void refuse(PyObject* type, const std::string& text) { throw Refused{type, text}; }

std::string str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(what) + ": a tensor is required");
  return THPVariable_Unpack(o);
}
bool none(PyObject* o) { return o == Py_None; }
bool truth(PyObject* o) {
  const int r = PyObject_IsTrue(o);
  if (r < 0) throw Refused{nullptr, ""};
  return r != 0;
}
int64_t whole(PyObject* o) {
  const int64_t r = PyLong_AsLongLong(o);
  if (r == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return r;
}
double real(PyObject* o) {
  const double r = PyFloat_AsDouble(o);
  if (r == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return r;
}
PyObject* item(PyObject* tuple, Py_ssize_t i, Py_ssize_t n, const char* what) {
  if (!PyTuple_Check(tuple) || PyTuple_GET_SIZE(tuple) != n) refuse(PyExc_TypeError, std::string(what) + ": a tuple of " + std::to_string(n) + " is required");
  return PyTuple_GET_ITEM(tuple, i);
}

// One call: the device it runs on, and the dtype code of its operands.
struct Call {
  int ordinal;
  bool amp;
  c10::cuda::OptionalCUDAGuard guard;
  Call(PyObject* ordinal_, PyObject* amp_) : ordinal((int)whole(ordinal_)), amp(truth(amp_)) {
    if (c10::cuda::current_device() != ordinal) guard.set_index((c10::DeviceIndex)ordinal);   // this device, whichever torch has made current
  }
  // Every operand on this device: the C ABI would read another device's memory, or the host's, as its own.
  void here(const at::Tensor& t) const {
    if (!t.is_cuda() || t.get_device() != ordinal)
      refuse(PyExc_ValueError, "a tensor on " + t.device().str() + ", the device is cuda:" + std::to_string(ordinal));
  }
  int dtype(const at::Tensor& t) const {
    if (t.scalar_type() == at::kHalf) return amp ? B200_AMP_F16 : B200_F16;
    if (t.scalar_type() == at::kFloat) return B200_F32;
    refuse(PyExc_TypeError, std::string("unsupported dtype ") + at::toString(t.scalar_type()) + ": f16 or f32 is required");
  }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, (c10::DeviceIndex)ordinal));
  }
  // A view shaped and typed like t that the caller gives, or a fresh contiguous tensor of that kind.
  at::Tensor like(PyObject* given, const at::Tensor& t, const char* what) const {
    if (none(given)) return empty(t.sizes(), t.scalar_type());
    const at::Tensor& g = tensor(given, what);
    if (g.sizes() != t.sizes() || g.scalar_type() != t.scalar_type())
      refuse(shape_mismatch, std::string(what) + ": " + str(g.sizes()) + " " + at::toString(g.scalar_type()) + ", " + str(t.sizes()) + " " +
                                 at::toString(t.scalar_type()) + " is required");
    here(g);
    return g;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)ordinal).stream(); }
};

void same_type(const at::Tensor& a, const at::Tensor& b) {
  if (a.scalar_type() != b.scalar_type())
    refuse(PyExc_TypeError, std::string(at::toString(a.scalar_type())) + " and " + at::toString(b.scalar_type()) + ": one type is required");
}

struct Strides {
  size_t s[4];
  explicit Strides(const at::Tensor& t) {
    for (int64_t i = 0; i < t.dim() && i < 4; ++i) s[i] = (size_t)t.stride(i);
  }
};

const int32_t* index(const Call& c, const at::Tensor& t, const char* what, at::IntArrayRef shape) {
  if (t.scalar_type() != at::kInt) refuse(PyExc_TypeError, std::string(what) + ": int32 is required, got " + at::toString(t.scalar_type()));
  if (t.sizes() != shape) refuse(shape_mismatch, std::string(what) + ": shape " + str(t.sizes()) + ", " + str(shape) + " is required");
  if (!t.is_contiguous()) refuse(PyExc_ValueError, std::string(what) + ": a contiguous tensor is required");
  c.here(t);
  return (const int32_t*)t.data_ptr();
}

// The words of a b200_head_op; returns the number of position axes that it reads.
int head_op(const Call& c, b200_head_op& op, int64_t d, const at::Tensor& like, PyObject* rotary, PyObject* norm, PyObject* q_gain,
            PyObject* k_gain, PyObject* eps) {
  op = {};
  int axes = 0;
  if (!none(rotary)) {
    const at::Tensor& f = tensor(item(rotary, 0, 3, "Rotary"), "Rotary.frequencies");
    PyObject* pairs = item(rotary, 1, 3, "Rotary");
    if (f.scalar_type() != at::kDouble || !f.is_contiguous()) refuse(PyExc_TypeError, "Rotary.frequencies: a contiguous f64 tensor is required");
    if (!PyTuple_Check(pairs) || PyTuple_GET_SIZE(pairs) < 1 || PyTuple_GET_SIZE(pairs) > 3)
      refuse(shape_mismatch, "Rotary.axis_pairs: one to three counts are required");
    int64_t all = 0;
    for (Py_ssize_t a = 0; a < PyTuple_GET_SIZE(pairs); ++a) {
      const int64_t n = whole(PyTuple_GET_ITEM(pairs, a));
      if (n < 0 || n > d) refuse(shape_mismatch, "Rotary.axis_pairs: " + std::to_string(n) + " pairs of heads of " + std::to_string(d));
      op.axis_pairs[a] = (size_t)n;
      all += n;
      if (n) axes = (int)a + 1;
    }
    if (f.numel() != all || 2 * all > d)
      refuse(shape_mismatch, "Rotary: " + std::to_string(f.numel()) + " frequencies for " + std::to_string(all) + " pairs of heads of " + std::to_string(d));
    c.here(f);
    op.frequencies = (const double*)f.data_ptr();
    op.interleaved = truth(item(rotary, 2, 3, "Rotary"));
  }
  op.normalize = truth(norm);
  op.epsilon = real(eps);
  PyObject* gains[2] = {q_gain, k_gain};
  for (int i = 0; i < 2; ++i) {
    if (none(gains[i])) continue;
    const at::Tensor& g = tensor(gains[i], "gain");
    if (!op.normalize) refuse(PyExc_ValueError, "a gain belongs to the norm");
    if (g.dim() != 1 || g.size(0) != d || g.scalar_type() != like.scalar_type() || !g.is_contiguous())
      refuse(shape_mismatch, "gain: " + std::to_string(d) + " contiguous elements of " + at::toString(like.scalar_type()) + " are required");
    c.here(g);
    (i ? op.k_gain : op.q_gain) = g.data_ptr();
  }
  return axes;
}

b200_kv_cache cache_of(const Call& c, PyObject* o) {
  const at::Tensor *k = &tensor(item(o, 0, 4, "cache"), "cache"), *v = &tensor(item(o, 1, 4, "cache"), "cache");
  const at::Tensor *ks = &tensor(item(o, 2, 4, "cache"), "cache"), *vs = &tensor(item(o, 3, 4, "cache"), "cache");
  const bool shaped = k->dim() == 4 && v->sizes() == k->sizes() && ks->dim() == 2 && vs->sizes() == ks->sizes() && ks->size(0) == k->size(0) &&
                      ks->size(1) == k->size(1);
  if (!shaped) refuse(shape_mismatch, "cache: codes " + str(k->sizes()) + ", " + str(v->sizes()) + ", scales " + str(ks->sizes()) + ", " + str(vs->sizes()));
  if (k->scalar_type() != at::kFloat8_e4m3fn || v->scalar_type() != at::kFloat8_e4m3fn || ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat)
    refuse(PyExc_TypeError, "cache: float8_e4m3fn codes and f32 scales are required");
  if (!k->is_contiguous() || !v->is_contiguous() || !ks->is_contiguous() || !vs->is_contiguous()) refuse(PyExc_ValueError, "cache: contiguous tensors are required");
  for (const at::Tensor* t : {k, v, ks, vs}) c.here(*t);
  return {k->data_ptr(), v->data_ptr(), (float*)ks->data_ptr(), (float*)vs->data_ptr(), (size_t)k->size(0), (size_t)k->size(1), (size_t)k->size(2), (size_t)k->size(3)};
}

b200_kv_batch batch_of(const Call& c, int64_t tokens, PyObject* cu_, PyObject* lens_, PyObject* table_, PyObject* max_new_) {
  const at::Tensor &cu = tensor(cu_, "cu_tokens"), &lens = tensor(lens_, "seq_lens"), &table = tensor(table_, "page_table");
  if (lens.dim() != 1) refuse(shape_mismatch, "seq_lens: one axis is required, got " + str(lens.sizes()));
  const int64_t n = lens.size(0), max_new = whole(max_new_);
  b200_kv_batch b;
  b.seqs = (size_t)n;
  b.tokens = (size_t)tokens;
  b.seq_lens = index(c, lens, "seq_lens", {n});
  b.cu_tokens = index(c, cu, "cu_tokens", {n + 1});
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != n)
    refuse(shape_mismatch, "page_table: int32 (" + std::to_string(n) + ", pages) is required, got " + at::toString(table.scalar_type()) + " " + str(table.sizes()));
  if (table.size(1) > 1 && table.stride(1) != 1) refuse(PyExc_ValueError, "page_table: a unit last stride is required");
  if (max_new < 0) refuse(shape_mismatch, "max_new: " + std::to_string(max_new));
  c.here(table);
  b.max_new = (size_t)std::min(max_new, tokens);
  b.page_table = (const int32_t*)table.data_ptr();
  b.page_table_stride = (size_t)(n > 1 ? table.stride(0) : table.size(1));
  b.max_pages = (size_t)table.size(1);
  return b;
}

// Raises what _lib.check makes of a status other than 0.
void checked(int status, const char* where) {
  if (status == B200_OK) return;
  PyObject* r = PyObject_CallFunction(check_status, "is", status, where);
  Py_XDECREF(r);
  throw Refused{nullptr, ""};
}

template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd are required", got, want);
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
    else if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "b200 call failed");
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// Hands over the references, also where one of the wraps fails.
PyObject* tuple_of(std::initializer_list<const at::Tensor*> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  Py_ssize_t i = 0;
  for (const at::Tensor* t : ts) {
    PyObject* o;
    if (r && t && t->defined()) {
      o = THPVariable_Wrap(*t);
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    if (!r || !o) {
      Py_XDECREF(o);
      Py_XDECREF(r);
      throw Refused{nullptr, ""};
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

void qk_shapes(const at::Tensor& q, const at::Tensor& k) {
  if (q.dim() != 4 || k.dim() != 4 || q.size(0) != k.size(0) || q.size(1) != k.size(1) || q.size(3) != k.size(3))
    refuse(shape_mismatch, "q " + str(q.sizes()) + ", k " + str(k.sizes()) + ": (batch, tokens, heads, d) each are required");
}

const int32_t* positions_of(const Call& c, PyObject* o, int axes, at::IntArrayRef rest) {
  if (none(o)) return nullptr;
  const at::Tensor& p = tensor(o, "positions");
  if (rest.size() == 2) return index(c, p, "positions", {std::max(axes, 1), rest[0], rest[1]});
  return index(c, p, "positions", {std::max(axes, 1), rest[0]});
}

// (ordinal, amp, q, k, rotary, positions, norm, q_gain, k_gain, eps, q_out, k_out)
PyObject* qk_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    Call c(a[0], a[1]);
    const at::Tensor &q = tensor(a[2], "q"), &k = tensor(a[3], "k");
    qk_shapes(q, k);
    same_type(q, k);
    const int dt = c.dtype(q);
    const int64_t b = q.size(0), s = q.size(1), hq = q.size(2), hk = k.size(2), d = q.size(3);
    b200_head_op op;
    const int axes = head_op(c, op, d, q, a[4], a[6], a[7], a[8], a[9]);
    const int32_t* pos = positions_of(c, a[5], axes, {b, s});
    c.here(q);
    c.here(k);
    const at::Tensor qo = c.like(a[10], q, "out"), ko = c.like(a[11], k, "out");
    const Strides qs(q), ks(k), qos(qo), kos(ko);
    void *stream = c.stream(), *qp = q.data_ptr(), *kp = k.data_ptr(), *qop = qo.data_ptr(), *kop = ko.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry.forward(dt, &op, b, s, hq, hk, d, qp, qs.s, kp, ks.s, pos, qop, qos.s, kop, kos.s, stream);
    Py_END_ALLOW_THREADS
    checked(rc, "b200_qk_norm_rotary_forward");
    return tuple_of({&qo, &ko});
  });
}

// (ordinal, amp, q, k, q_grad_out, k_grad_out, rotary, positions, norm, q_gain, k_gain, eps, grad_q, grad_k, q_gain_grad, k_gain_grad)
PyObject* qk_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    Call c(a[0], a[1]);
    const at::Tensor &q = tensor(a[2], "q"), &k = tensor(a[3], "k");
    at::Tensor gq = tensor(a[4], "grad_q_out"), gk = tensor(a[5], "grad_k_out");
    qk_shapes(q, k);
    if (gq.sizes() != q.sizes() || gk.sizes() != k.sizes()) refuse(shape_mismatch, "upstream gradients shaped like q and k are required");
    same_type(q, k);
    same_type(q, gq);
    same_type(q, gk);
    const int dt = c.dtype(q);
    const int64_t b = q.size(0), s = q.size(1), hq = q.size(2), hk = k.size(2), d = q.size(3);
    b200_head_op op;
    const int axes = head_op(c, op, d, q, a[6], a[8], a[9], a[10], a[11]);
    const int32_t* pos = positions_of(c, a[7], axes, {b, s});
    for (const at::Tensor* t : {&q, &k, (const at::Tensor*)&gq, (const at::Tensor*)&gk}) c.here(*t);
    if (gq.stride(3) != 1) gq = gq.contiguous();
    if (gk.stride(3) != 1) gk = gk.contiguous();
    const at::Tensor dq = c.like(a[12], q, "out"), dk = c.like(a[13], k, "out");
    at::Tensor sums, dqg, dkg, ws;
    size_t need = 0;
    const bool add = !none(a[14]);
    if (op.normalize) {
      if (add) {
        dqg = tensor(a[14], "gain_grads");
        dkg = tensor(a[15], "gain_grads");
        for (const at::Tensor* t : {&dqg, &dkg}) {
          if (t->scalar_type() != at::kFloat || t->dim() != 1 || t->size(0) != d || !t->is_contiguous())
            refuse(shape_mismatch, "gain_grads: two f32 tensors of " + std::to_string(d) + " elements are required");
          c.here(*t);
        }
      } else {
        dqg = c.empty({d}, at::kFloat);
        dkg = c.empty({d}, at::kFloat);
      }
      // from torch's allocator rather than the device's one workspace: calls on several streams, and graphs, have their own
      need = entry.backward_bytes((size_t)d);
      ws = c.empty({(int64_t)need}, at::kByte);
    }
    const Strides qs(q), ks(k), gqs(gq), gks(gk), dqs(dq), dks(dk);
    void *stream = c.stream(), *p[6] = {q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr()};
    float *pg[2] = {dqg.defined() ? (float*)dqg.data_ptr() : nullptr, dkg.defined() ? (float*)dkg.data_ptr() : nullptr};
    void* pw = ws.defined() ? ws.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry.backward(dt, &op, b, s, hq, hk, d, p[0], qs.s, p[1], ks.s, pos, p[2], gqs.s, p[3], gks.s, p[4], dqs.s, p[5], dks.s, pg[0], pg[1], add, pw,
                        need, stream);
    Py_END_ALLOW_THREADS
    checked(rc, "b200_qk_norm_rotary_backward");
    return tuple_of({&dq, &dk, &dqg, &dkg});
  });
}

// (ordinal, amp, cache, k, v, cu_tokens, seq_lens, page_table, max_new, q, rotary, positions, norm, q_gain, k_gain, eps, q_out)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 17, [&]() -> PyObject* {
    Call c(a[0], a[1]);
    const b200_kv_cache cache = cache_of(c, a[2]);
    const at::Tensor &k = tensor(a[3], "k"), &v = tensor(a[4], "v");
    const bool has_q = !none(a[9]);
    const at::Tensor* q = has_q ? &tensor(a[9], "q") : nullptr;
    const int64_t d = (int64_t)cache.d;
    const bool shaped = k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == (int64_t)cache.heads && k.size(2) == d &&
                        (!q || (q->dim() == 3 && q->size(0) == k.size(0) && q->size(2) == d));
    if (!shaped)
      refuse(shape_mismatch, "k " + str(k.sizes()) + ", v " + str(v.sizes()) + ", q " + (q ? str(q->sizes()) : "None") + ": (tokens, heads, " + std::to_string(d) +
                                 ") with the cache's " + std::to_string(cache.heads) + " key heads are required");
    same_type(k, v);
    if (q) same_type(k, *q);
    const int dt = c.dtype(k);
    const int64_t t = k.size(0);
    b200_head_op op;
    const int axes = head_op(c, op, d, k, a[10], a[12], a[13], a[14], a[15]);
    const int32_t* pos = positions_of(c, a[11], axes, {t});
    const b200_kv_batch batch = batch_of(c, t, a[5], a[6], a[7], a[8]);
    c.here(k);
    c.here(v);
    if (q) c.here(*q);
    at::Tensor qo;
    if (q) qo = c.like(a[16], *q, "q_out");
    const Strides ks(k), vs(v), qs(q ? *q : k), qos(q ? qo : k);
    void *stream = c.stream(), *kp = k.data_ptr(), *vp = v.data_ptr(), *qp = q ? q->data_ptr() : nullptr, *qop = q ? qo.data_ptr() : nullptr;
    const size_t hq = q ? (size_t)q->size(1) : 0;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry.append(dt, &cache, &batch, &op, hq, qp, qs.s, kp, ks.s, vp, vs.s, pos, qop, qos.s, stream);
    Py_END_ALLOW_THREADS
    checked(rc, "b200_kv_cache_append");
    if (!q) Py_RETURN_NONE;
    return THPVariable_Wrap(qo);
  });
}

// (ordinal, cache, pages, f16)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    Call c(a[0], Py_False);
    const b200_kv_cache cache = cache_of(c, a[1]);
    const at::Tensor& pages = tensor(a[2], "pages");
    if (pages.dim() != 1) refuse(shape_mismatch, "pages: one axis is required, got " + str(pages.sizes()));
    const int64_t m = pages.size(0);
    const int32_t* ids = index(c, pages, "pages", {m});
    const bool half = truth(a[3]);
    const int64_t shape[4] = {m, (int64_t)cache.heads, (int64_t)cache.page_size, (int64_t)cache.d};
    const at::Tensor k = c.empty(shape, half ? at::kHalf : at::kFloat), v = c.empty(shape, half ? at::kHalf : at::kFloat);
    void *stream = c.stream(), *kp = k.data_ptr(), *vp = v.data_ptr();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry.read(half ? B200_F16 : B200_F32, &cache, (size_t)m, ids, kp, vp, stream);
    Py_END_ALLOW_THREADS
    checked(rc, "b200_kv_cache_read");
    return tuple_of({&k, &v});
  });
}

// (ordinal, amp, cache, q, cu_tokens, seq_lens, page_table, max_new, alpha, causal, window, out, want_lse)
PyObject* kv_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    Call c(a[0], a[1]);
    const b200_kv_cache cache = cache_of(c, a[2]);
    const at::Tensor& q = tensor(a[3], "q");
    if (q.dim() != 3 || q.size(2) != (int64_t)cache.d || cache.heads == 0 || q.size(1) % (int64_t)cache.heads)
      refuse(shape_mismatch, "q " + str(q.sizes()) + ": (tokens, a multiple of " + std::to_string(cache.heads) + " heads, " + std::to_string(cache.d) + ") is required");
    const int dt = c.dtype(q), causal = truth(a[9]);
    const int64_t t = q.size(0), hq = q.size(1), window = whole(a[10]);
    const double alpha = real(a[8]);
    if (window < 0) refuse(shape_mismatch, "window: " + std::to_string(window));
    const b200_kv_batch batch = batch_of(c, t, a[4], a[5], a[6], a[7]);
    c.here(q);
    const at::Tensor out = c.like(a[11], q, "out");
    at::Tensor lse, ws;
    if (truth(a[12])) lse = c.empty({t, hq}, at::kFloat);
    // from torch's allocator rather than the device's one workspace: calls on several streams, and graphs, have their own
    const size_t need = entry.attention_bytes(&cache, &batch, (size_t)hq, causal, (size_t)window);
    if (need) ws = c.empty({(int64_t)need}, at::kByte);
    const Strides qs(q), os(out);
    void *stream = c.stream(), *qp = q.data_ptr(), *op = out.data_ptr(), *wp = need ? ws.data_ptr() : nullptr;
    float* lp = lse.defined() ? (float*)lse.data_ptr() : nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = entry.attention(dt, &cache, &batch, (size_t)hq, qp, qs.s, alpha, causal, (size_t)window, op, os.s, lp, wp, need, stream);
    Py_END_ALLOW_THREADS
    checked(rc, "b200_kv_cache_attention");
    return tuple_of({&out, &lse});
  });
}

// (ShapeMismatch, check, addresses of the seven entry points in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    void* p[7];
    for (int i = 0; i < 7; ++i) p[i] = (void*)(uintptr_t)whole(a[2 + i]);
    entry.forward = (decltype(entry.forward))p[0];
    entry.backward = (decltype(entry.backward))p[1];
    entry.backward_bytes = (decltype(entry.backward_bytes))p[2];
    entry.append = (decltype(entry.append))p[3];
    entry.read = (decltype(entry.read))p[4];
    entry.attention = (decltype(entry.attention))p[5];
    entry.attention_bytes = (decltype(entry.attention_bytes))p[6];
    Py_INCREF(a[0]);
    Py_INCREF(a[1]);
    Py_XSETREF(shape_mismatch, a[0]);
    Py_XSETREF(check_status, a[1]);
    Py_RETURN_NONE;
  });
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(bind), FAST(qk_forward), FAST(qk_backward), FAST(kv_append), FAST(kv_read), FAST(kv_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_heads", "Host side of dfdx_b200.heads.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__heads(void) { return PyModule_Create(&module); }
