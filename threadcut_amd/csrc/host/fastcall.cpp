// The call paths of a decode step in native code: what the Python wrappers do
// per call (tensor checks, stride arrays, workspace, the library call) for the
// calls that need no special treatment, without ctypes.
//
// Each function returns None (or False) for anything else: another device
// than the current one, a tensor subclass, a shape, type or stride that the
// kernels refuse. The Python wrapper then takes the call, checks it in full
// and raises what there is to raise. Nothing is enqueued in that case: the
// library validates before it launches.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/InferenceMode.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <vector>

#include "../../../include/threadcut_hip.h"

namespace {

constexpr int64_t kHeadDim = 128;

bool dtype_code(const at::Tensor& t, int* code) {
  if (t.scalar_type() == at::kHalf) { *code = TC_DTYPE_F16; return true; }
  if (t.scalar_type() == at::kBFloat16) { *code = TC_DTYPE_BF16; return true; }
  return false;
}

// A plain torch.Tensor with memory on the current GPU. The device is looked
// up once per call and passed on.
const at::Tensor* tensor(PyObject* o, const c10::Device& dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.has_storage() || t.device() != dev || t.layout() != at::kStrided) return nullptr;
  return &t;
}

bool current(PyObject* o, c10::Device* dev) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda()) return false;
  const c10::impl::DeviceGuardImplInterface* impl = c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA);
  *dev = t.device();
  return impl->getDevice() == *dev;
}

int64_t stride(const at::Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; }

// The cache's [B, Hkv, N, 128] strides; a single token's row keeps its own length.
void cache_strides(const at::Tensor& t, int64_t st[3]) {
  st[0] = stride(t, 0);
  st[1] = stride(t, 1);
  st[2] = t.size(2) > 1 ? t.stride(2) : kHeadDim;
}

bool same_type(const at::Tensor& q, const at::Tensor& t) { return t.scalar_type() == q.scalar_type(); }

// q [B, Hq, 1, 128] of a decode step with its KV heads: batch, heads, group
// and the strides of its [B, Hkv, G, 128] view.
struct Query {
  int64_t b, hq, hkv, g;
  int64_t st[3];
  int dt;
};

bool query(const at::Tensor& q, const at::Tensor& k, Query* x) {
  if (q.dim() != 4 || k.dim() != 4 || q.size(2) != 1 || q.size(3) != kHeadDim || k.size(3) != kHeadDim) return false;
  if (!dtype_code(q, &x->dt) || !same_type(q, k) || q.stride(3) != 1 || k.stride(3) != 1) return false;
  x->b = q.size(0);
  x->hq = q.size(1);
  x->hkv = k.size(1);
  if (x->b < 1 || k.size(0) != x->b || x->hkv < 1 || x->hq % x->hkv) return false;
  x->g = x->hq / x->hkv;
  if (x->g < 1 || x->g > 8) return false;
  const int64_t sh = q.stride(1);
  x->st[0] = stride(q, 0);
  x->st[1] = x->hkv > 1 ? x->g * sh : 0;
  x->st[2] = x->g > 1 ? sh : 0;
  return true;
}

// The split plan's workspace; false for a plan that the library refuses.
bool workspace(const at::Tensor& q, const Query& x, int64_t n, int64_t split, int ragged, at::Tensor* ws) {
  const int s = tc_decode_num_splits(static_cast<int>(x.b), static_cast<int>(x.hkv), n, static_cast<int>(split), ragged);
  if (s < 0) return false;
  const size_t bytes = tc_decode_workspace_bytes(static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g),
                                                 static_cast<int>(kHeadDim), s);
  *ws = at::empty({static_cast<int64_t>(bytes < 16 ? 16 : bytes)}, q.options().dtype(at::kByte).requires_grad(false));
  return true;
}

// The output [B, 1, Hq, 128] and its strides as [B, Hkv, G, 128].
at::Tensor output(const at::Tensor& q, const Query& x, int64_t st[3]) {
  st[0] = x.hq * kHeadDim;
  st[1] = x.g * kHeadDim;
  st[2] = kHeadDim;
  return at::empty({x.b, 1, x.hq, kHeadDim}, q.options().requires_grad(false));
}

void* raw_stream(PyObject* o) { return reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o))); }

// A new token's rows [B, Hkv, 128] or [B, Hkv, 1, 128] and their (batch, head) strides.
bool new_rows(const at::Tensor& t, const at::Tensor& q, const Query& x, int64_t st[2]) {
  if (!same_type(q, t) || (t.dim() != 3 && !(t.dim() == 4 && t.size(2) == 1))) return false;
  if (t.size(0) != x.b || t.size(1) != x.hkv || t.size(-1) != kHeadDim || t.stride(-1) != 1) return false;
  st[0] = stride(t, 0);
  st[1] = stride(t, 1);
  return true;
}

// A sliding window that hides some of n tokens (0: none does); false for one that the library refuses.
struct Window {
  int64_t size = 0, sinks = 0, span = 0;  // span: the tokens that the split plan is made for
};

bool window(PyObject* size, PyObject* sinks, int64_t n, Window* w) {
  if (size == Py_None) return true;
  const int64_t x = PyLong_AsLongLong(size), y = PyLong_AsLongLong(sinks);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  const int64_t span = tc_decode_window_tokens(n, x, y);
  if (span < 0) return false;
  if (x < n && n - x > y) *w = Window{x, y, span};
  return true;
}

// decode(query [b, hq, 1, d], key, value [b, hkv, n, d], scale, stream[, window, sinks]) -> out [b, 1, hq, d] or None
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if ((n_args != 5 && n_args != 7) || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0], dev), *k = tensor(a[1], dev), *v = tensor(a[2], dev);
  Query x;
  if (!q || !k || !v || !query(*q, *k, &x)) Py_RETURN_NONE;
  if (!same_type(*q, *v) || v->sizes() != k->sizes() || v->stride(3) != 1) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[3]);
  void* stream = raw_stream(a[4]);
  if (PyErr_Occurred()) return nullptr;
  int64_t so[3], sk[3], sv[3];
  cache_strides(*k, sk);
  cache_strides(*v, sv);
  const int64_t n = k->size(2);
  Window w;
  if (n_args == 7 && !window(a[5], a[6], n, &w)) Py_RETURN_NONE;
  at::Tensor ws;
  if (!workspace(*q, x, w.size ? w.span : n, 0, 0, &ws)) Py_RETURN_NONE;
  at::Tensor out = output(*q, x, so);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (w.size)
    rc = tc_decode_window_attention(q->const_data_ptr(), x.st, k->const_data_ptr(), sk, v->const_data_ptr(), sv, nullptr,
                                    n, w.size, w.sinks, static_cast<int>(x.b), static_cast<int>(x.hkv),
                                    static_cast<int>(x.g), kHeadDim, x.dt, static_cast<float>(scale), 0,
                                    ws.mutable_data_ptr(), ws.numel(), out.mutable_data_ptr(), so, stream);
  else
    rc = tc_decode_attention(q->const_data_ptr(), x.st, k->const_data_ptr(), sk, v->const_data_ptr(), sv, nullptr, n,
                             static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g), kHeadDim, x.dt,
                             static_cast<float>(scale), 0, ws.mutable_data_ptr(), ws.numel(), out.mutable_data_ptr(),
                             so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// decode_append(query, k_buf, v_buf [b, hkv, cap, d], k_new, v_new, n or pos, scale, stream[, window, sinks]) -> out or
// None.
// A whole number: the rows go to token n - 1; an int32 [b] tensor: to token pos[b] (the plan is the capacity's).
PyObject* decode_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if ((n_args != 8 && n_args != 10) || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0], dev), *k = tensor(a[1], dev), *v = tensor(a[2], dev), *kn = tensor(a[3], dev),
                   *vn = tensor(a[4], dev);
  Query x;
  int64_t so[3], sk[3], sv[3], skn[2], svn[2];
  if (!q || !k || !v || !kn || !vn || !query(*q, *k, &x)) Py_RETURN_NONE;
  if (!same_type(*q, *v) || v->sizes() != k->sizes() || v->stride(3) != 1) Py_RETURN_NONE;
  if (!new_rows(*kn, *q, x, skn) || !new_rows(*vn, *q, x, svn)) Py_RETURN_NONE;
  const int64_t cap = k->size(2);
  const int32_t* pos = nullptr;
  int64_t n = cap;
  if (THPVariable_Check(a[5])) {
    const at::Tensor* p = tensor(a[5], dev);
    if (!p || p->scalar_type() != at::kInt || p->dim() != 1 || p->size(0) != x.b || !p->is_contiguous()) Py_RETURN_NONE;
    pos = static_cast<const int32_t*>(p->const_data_ptr());
  } else {
    n = PyLong_AsLongLong(a[5]);
  }
  const double scale = PyFloat_AsDouble(a[6]);
  void* stream = raw_stream(a[7]);
  if (PyErr_Occurred()) return nullptr;
  if (n < 1 || n > cap) Py_RETURN_NONE;
  cache_strides(*k, sk);
  cache_strides(*v, sv);
  Window w;
  if (n_args == 10 && !window(a[8], a[9], n, &w)) Py_RETURN_NONE;
  at::Tensor ws;
  if (!workspace(*q, x, w.size ? w.span : n, 0, 0, &ws)) Py_RETURN_NONE;
  at::Tensor out = output(*q, x, so);
  const int b = static_cast<int>(x.b), hkv = static_cast<int>(x.hkv), g = static_cast<int>(x.g);
  const float sc = static_cast<float>(scale);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (w.size)
    rc = tc_decode_append_window_attention(q->const_data_ptr(), x.st, k->mutable_data_ptr(), sk, v->mutable_data_ptr(),
                                           sv, kn->const_data_ptr(), skn, vn->const_data_ptr(), svn, pos, n, w.size,
                                           w.sinks, b, hkv, g, kHeadDim, x.dt, sc, 0, ws.mutable_data_ptr(), ws.numel(),
                                           out.mutable_data_ptr(), so, stream);
  else
    rc = pos ? tc_decode_append_attention_at(q->const_data_ptr(), x.st, k->mutable_data_ptr(), sk,
                                             v->mutable_data_ptr(), sv, kn->const_data_ptr(), skn, vn->const_data_ptr(),
                                             svn, pos, cap, b, hkv, g, kHeadDim, x.dt, sc, 0, ws.mutable_data_ptr(),
                                             ws.numel(), out.mutable_data_ptr(), so, stream)
             : tc_decode_append_attention(q->const_data_ptr(), x.st, k->mutable_data_ptr(), sk, v->mutable_data_ptr(),
                                          sv, kn->const_data_ptr(), skn, vn->const_data_ptr(), svn, n, b, hkv, g,
                                          kHeadDim, x.dt, sc, 0, ws.mutable_data_ptr(), ws.numel(),
                                          out.mutable_data_ptr(), so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_append(q [b, hkv, g, d], k_pool, v_pool [pages, hkv, P, d], table [b, tiles, 4], counts [b], k_new, v_new,
// out or None, scale, stream) -> out [b, hkv, g, d] or None: PagedKV.decode_append's call.
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 10 || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor* t[7];
  for (int i = 0; i < 7; ++i)
    if (!(t[i] = tensor(a[i], dev))) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &tab = *t[3], &cnt = *t[4], &kn = *t[5], &vn = *t[6];
  Query x;
  if (q.dim() != 4 || kp.dim() != 4 || q.size(3) != kHeadDim || kp.size(3) != kHeadDim || !dtype_code(q, &x.dt)) Py_RETURN_NONE;
  if (!same_type(q, kp) || !same_type(q, vp) || vp.sizes() != kp.sizes() || vp.strides() != kp.strides()) Py_RETURN_NONE;
  x.b = q.size(0);
  x.hkv = q.size(1);
  x.g = q.size(2);
  if (x.b < 1 || kp.size(1) != x.hkv || q.stride(3) != 1 || kp.stride(3) != 1 || tab.dim() != 3 || tab.size(0) != x.b) Py_RETURN_NONE;
  int64_t skn[2], svn[2];
  if (!new_rows(kn, q, x, skn) || !new_rows(vn, q, x, svn)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[8]);
  void* stream = raw_stream(a[9]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out;
  if (a[7] == Py_None) {
    out = at::empty_like(q);
  } else {
    const at::Tensor* o = tensor(a[7], dev);
    if (!o || o->sizes() != q.sizes() || !same_type(q, *o) || o->stride(3) != 1) Py_RETURN_NONE;
    out = *o;
  }
  const int64_t tiles = tab.size(1);
  at::Tensor ws;
  if (!workspace(q, x, 16 * tiles, 0, x.b > 1, &ws)) Py_RETURN_NONE;
  const int64_t sq[3] = {q.stride(0), q.stride(1), q.stride(2)}, sp[3] = {kp.stride(0), kp.stride(1), kp.stride(2)},
                so[3] = {out.stride(0), out.stride(1), out.stride(2)};
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_decode_paged_append_attention(
      q.const_data_ptr(), sq, kp.mutable_data_ptr(), vp.mutable_data_ptr(), sp, static_cast<int>(kp.size(0)),
      static_cast<int>(kp.size(2)), static_cast<const int32_t*>(tab.const_data_ptr()),
      static_cast<const int32_t*>(cnt.const_data_ptr()), tiles, kn.const_data_ptr(), skn, vn.const_data_ptr(), svn,
      static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g), kHeadDim, x.dt, static_cast<float>(scale), 0,
      ws.mutable_data_ptr(), ws.numel(), out.mutable_data_ptr(), so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// q [b, hkv, g, d] of a call with grouped queries, and where its output goes: `o`, or a new tensor.
bool grouped(const at::Tensor& q, Query* x) {
  if (q.dim() != 4 || q.size(3) != kHeadDim || q.stride(3) != 1 || !dtype_code(q, &x->dt)) return false;
  x->b = q.size(0);
  x->hkv = q.size(1);
  x->g = q.size(2);
  x->hq = x->hkv * x->g;
  for (int i = 0; i < 3; ++i) x->st[i] = stride(q, i);
  return x->b >= 1;
}

bool grouped_out(PyObject* o, const at::Tensor& q, const c10::Device& dev, at::Tensor* out, int64_t st[3]) {
  if (o == Py_None) {
    *out = at::empty(q.sizes(), q.options().requires_grad(false));
  } else {
    const at::Tensor* t = tensor(o, dev);
    if (!t || t->sizes() != q.sizes() || !same_type(q, *t) || t->stride(3) != 1) return false;
    *out = *t;
  }
  for (int i = 0; i < 3; ++i) st[i] = stride(*out, i);
  return true;
}

// Pools [pages, hkv, P, d] of one layer that fit the query.
bool pools(const at::Tensor& q, const Query& x, const at::Tensor& kp, const at::Tensor& vp, int64_t st[3]) {
  if (kp.dim() != 4 || kp.size(1) != x.hkv || kp.size(3) != kHeadDim || kp.stride(3) != 1 || !same_type(q, kp) ||
      !same_type(q, vp) || vp.sizes() != kp.sizes() || vp.strides() != kp.strides())
    return false;
  for (int i = 0; i < 3; ++i) st[i] = kp.stride(i);
  return true;
}

// int32 tables, contiguous (an empty one has no address).
bool table(const at::Tensor& t) { return t.scalar_type() == at::kInt && t.is_contiguous(); }
const int32_t* words(const at::Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }

// paged_decode(q [b, hkv, g, d], k_pool, v_pool, table [b, tiles, 4], counts [b], out or None, scale, stream) -> out or
// None: PagedKV.decode's call.
PyObject* paged_decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 8 || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i)
    if (!(t[i] = tensor(a[i], dev))) Py_RETURN_NONE;
  Query x;
  int64_t sp[3], so[3];
  if (!grouped(*t[0], &x) || !pools(*t[0], x, *t[1], *t[2], sp)) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &tab = *t[3], &cnt = *t[4];
  if (tab.dim() != 3 || tab.size(0) != x.b || !table(tab) || cnt.numel() != x.b || !table(cnt)) Py_RETURN_NONE;
  at::Tensor out, ws;
  if (!grouped_out(a[5], q, dev, &out, so)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[6]);
  void* stream = raw_stream(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t tiles = tab.size(1);
  if (!workspace(q, x, 16 * tiles, 0, x.b > 1, &ws)) Py_RETURN_NONE;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_decode_paged_attention(q.const_data_ptr(), x.st, kp.const_data_ptr(), vp.const_data_ptr(), sp,
                                 static_cast<int>(kp.size(0)), static_cast<int>(kp.size(2)), words(tab), words(cnt),
                                 tiles, static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g), kHeadDim,
                                 x.dt, static_cast<float>(scale), 0, ws.mutable_data_ptr(), ws.numel(),
                                 out.mutable_data_ptr(), so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The workspace of a shared-prefix call.
bool shared_workspace(const at::Tensor& q, const Query& x, int64_t prefix, int64_t n, int ragged, at::Tensor* ws) {
  const int s = tc_decode_shared_num_splits(static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g), prefix,
                                            n, ragged);
  if (s < 0) return false;
  const size_t bytes = tc_decode_workspace_bytes(static_cast<int>(x.b), static_cast<int>(x.hkv), static_cast<int>(x.g),
                                                 static_cast<int>(kHeadDim), s);
  *ws = at::empty({static_cast<int64_t>(bytes < 16 ? 16 : bytes)}, q.options().dtype(at::kByte).requires_grad(false));
  return true;
}

// paged_shared(q [b, hkv, g, d], k_pool, v_pool, shared table [T, 4], table [b, tiles, 4], counts [b], k_new, v_new (or
// None), out or None, scale, stream) -> out or None: PagedKV's calls on forked sequences.
PyObject* paged_shared(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 11 || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = tensor(a[i], dev))) Py_RETURN_NONE;
  Query x;
  int64_t sp[3], so[3], skn[2] = {0, 0}, svn[2] = {0, 0};
  if (!grouped(*t[0], &x) || !pools(*t[0], x, *t[1], *t[2], sp)) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &head = *t[3], &tab = *t[4], &cnt = *t[5];
  if (head.dim() != 2 || !table(head) || tab.dim() != 3 || tab.size(0) != x.b || !table(tab) || cnt.numel() != x.b ||
      !table(cnt))
    Py_RETURN_NONE;
  const at::Tensor *kn = nullptr, *vn = nullptr;
  if (a[6] != Py_None) {
    kn = tensor(a[6], dev);
    vn = tensor(a[7], dev);
    if (!kn || !vn || !new_rows(*kn, q, x, skn) || !new_rows(*vn, q, x, svn)) Py_RETURN_NONE;
  }
  at::Tensor out, ws;
  if (!grouped_out(a[8], q, dev, &out, so)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[9]);
  void* stream = raw_stream(a[10]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t shared = head.size(0), tiles = tab.size(1);
  if (!shared_workspace(q, x, 16 * shared, 16 * tiles, x.b > 1, &ws)) Py_RETURN_NONE;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_decode_paged_shared_attention(
      q.const_data_ptr(), x.st, kp.mutable_data_ptr(), vp.mutable_data_ptr(), sp, static_cast<int>(kp.size(0)),
      static_cast<int>(kp.size(2)), words(head), shared, words(tab), words(cnt), tiles,
      kn ? kn->const_data_ptr() : nullptr, skn, vn ? vn->const_data_ptr() : nullptr, svn, static_cast<int>(x.b),
      static_cast<int>(x.hkv), static_cast<int>(x.g), kHeadDim, x.dt, static_cast<float>(scale), ws.mutable_data_ptr(),
      ws.numel(), out.mutable_data_ptr(), so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// decode_shared(q [b, hkv, g, d], k_prefix, v_prefix [hkv, p, d] or [1, hkv, p, d], k, v [b, hkv, n, d], lens [b] or
// None, out or None, scale, stream) -> out or None
PyObject* decode_shared(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 9 || !current(a[0], &dev)) Py_RETURN_NONE;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i)
    if (!(t[i] = tensor(a[i], dev))) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &kp = *t[1], &vp = *t[2], &k = *t[3], &v = *t[4];
  Query x;
  if (!grouped(q, &x) || k.dim() != 4 || v.sizes() != k.sizes() || k.size(0) != x.b || k.size(1) != x.hkv) Py_RETURN_NONE;
  if (vp.sizes() != kp.sizes() || (kp.dim() != 3 && !(kp.dim() == 4 && kp.size(0) == 1))) Py_RETURN_NONE;
  const int at = kp.dim() - 3;
  if (kp.size(at) != x.hkv) Py_RETURN_NONE;
  for (int i = 1; i < 5; ++i)
    if (!same_type(q, *t[i]) || t[i]->size(-1) != kHeadDim || t[i]->stride(-1) != 1) Py_RETURN_NONE;
  const int32_t* lens = nullptr;
  if (a[5] != Py_None) {
    const at::Tensor* l = tensor(a[5], dev);
    if (!l || l->dim() != 1 || l->size(0) != x.b || !table(*l)) Py_RETURN_NONE;
    lens = words(*l);
  }
  at::Tensor out, ws;
  int64_t so[3], sk[3], sv[3];
  if (!grouped_out(a[6], q, dev, &out, so)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[7]);
  void* stream = raw_stream(a[8]);
  if (PyErr_Occurred()) return nullptr;
  cache_strides(k, sk);
  cache_strides(v, sv);
  const int64_t prefix = kp.size(at + 1), n = k.size(2);
  auto head_token = [&](const at::Tensor& p, int64_t st[2]) {
    st[0] = stride(p, at);
    st[1] = prefix > 1 ? p.stride(at + 1) : kHeadDim;
  };
  int64_t skp[2], svp[2];
  head_token(kp, skp);
  head_token(vp, svp);
  if (!shared_workspace(q, x, prefix, n, lens != nullptr, &ws)) Py_RETURN_NONE;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_decode_shared_attention(q.const_data_ptr(), x.st, kp.const_data_ptr(), skp, vp.const_data_ptr(), svp, prefix,
                                  k.const_data_ptr(), sk, v.const_data_ptr(), sv, lens, n, static_cast<int>(x.b),
                                  static_cast<int>(x.hkv), static_cast<int>(x.g), kHeadDim, x.dt,
                                  static_cast<float>(scale), ws.mutable_data_ptr(), ws.numel(), out.mutable_data_ptr(),
                                  so, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// True for a tensor whose in-place copy torch would record or refuse: autograd (a view of a tracked buffer counts),
// a forward-mode tangent, an inference tensor outside inference mode.
bool recorded(const at::Tensor& t) {
  return (c10::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined() ||
         (t.is_inference() && !c10::InferenceMode::is_enabled());
}

// True while something sees every operation of this thread: torch.jit.trace, a dispatch mode and a functorch transform
// each include a dispatch key of their own.
bool watched() {
  return !(c10::impl::tls_local_dispatch_key_set().included_ - c10::default_included_set).empty();
}

// append_rows(k_buf, v_buf [b, h, cap, d], row0, k, v [b, h, rows, d], stream) -> bool: new tokens' rows into both
// buffers. Autograd is told of the write (the buffers' versions), as torch's copy would tell it.
PyObject* append_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 6 || !current(a[0], &dev)) Py_RETURN_FALSE;
  const at::Tensor *kb = tensor(a[0], dev), *vb = tensor(a[1], dev), *k = tensor(a[3], dev), *v = tensor(a[4], dev);
  int dt;
  if (!kb || !vb || !k || !v || kb->dim() != 4 || k->dim() != 4 || !dtype_code(*kb, &dt)) Py_RETURN_FALSE;
  if (vb->sizes() != kb->sizes() || vb->strides() != kb->strides() || v->sizes() != k->sizes()) Py_RETURN_FALSE;
  for (const at::Tensor* t : {k, v})
    if (!same_type(*kb, *t) || t->size(0) != kb->size(0) || t->size(1) != kb->size(1) || t->size(3) != kHeadDim ||
        kb->size(3) != kHeadDim || t->stride(3) != 1)
      Py_RETURN_FALSE;
  // Writes that autograd, tracing, a dispatch mode or a functorch transform would record stay torch's copies.
  for (const at::Tensor* t : {kb, vb, k, v})
    if (recorded(*t)) Py_RETURN_FALSE;
  if (watched()) Py_RETURN_FALSE;
  const int64_t row0 = PyLong_AsLongLong(a[2]);
  void* stream = raw_stream(a[5]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t sk[3] = {k->stride(0), k->stride(1), k->stride(2)}, sv[3] = {v->stride(0), v->stride(1), v->stride(2)},
                sb[3] = {kb->stride(0), kb->stride(1), kb->stride(2)};
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_append_rows(k->const_data_ptr(), sk, v->const_data_ptr(), sv, kb->mutable_data_ptr(), vb->mutable_data_ptr(),
                      sb, kb->size(2), row0, static_cast<int>(kb->size(0)), static_cast<int>(kb->size(1)), k->size(2),
                      kHeadDim, dt, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_FALSE;
  if (!kb->is_inference()) kb->unsafeGetTensorImpl()->bump_version();
  if (!vb->is_inference()) vb->unsafeGetTensorImpl()->bump_version();
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// The tensors of one of rope_rows' lists: plain rows [b, h, n, d] (or [h, n, d] of one sequence, [b, h, d] of one
// token) of one set of strides, that torch's copy would not record.
bool row_list(PyObject* list, const c10::Device& dev, at::ScalarType type, int64_t b, int64_t n, int64_t* heads,
              std::vector<const void*>* ptrs, int64_t st[3]) {
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(list);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor* t = tensor(PySequence_Fast_GET_ITEM(list, i), dev);
    if (!t || t->scalar_type() != type || t->size(-1) != kHeadDim || t->stride(-1) != 1 || recorded(*t)) return false;
    int64_t s[3], h;
    if (t->dim() == 4 && t->size(0) == b && t->size(2) == n) {
      h = t->size(1);
      for (int j = 0; j < 3; ++j) s[j] = stride(*t, j);
    } else if (t->dim() == 3 && b == 1 && t->size(1) == n) {
      h = t->size(0);
      s[0] = 0; s[1] = stride(*t, 0); s[2] = stride(*t, 1);
    } else if (t->dim() == 3 && n == 1 && t->size(0) == b) {
      h = t->size(1);
      s[0] = stride(*t, 0); s[1] = stride(*t, 1); s[2] = 0;
    } else {
      return false;
    }
    if (i == 0) {
      *heads = h;
      for (int j = 0; j < 3; ++j) st[j] = s[j];
    }
    if (h != *heads || s[0] != st[0] || s[1] != st[1] || s[2] != st[2]) return false;
    ptrs->push_back(t->const_data_ptr());
  }
  return true;
}

bool pool_list(PyObject* list, const c10::Device& dev, const at::Tensor& like, std::vector<void*>* ptrs) {
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(list);
  for (Py_ssize_t i = 0; i < count; ++i) {
    const at::Tensor* t = tensor(PySequence_Fast_GET_ITEM(list, i), dev);
    if (!t || t->scalar_type() != like.scalar_type() || t->sizes() != like.sizes() || t->strides() != like.strides() ||
        recorded(*t))
      return false;
    ptrs->push_back(t->mutable_data_ptr());
  }
  return true;
}

// rope_rows(k rows, v rows, k pools, v pools (a list or tuple of each, one per layer), slots [b, n, 4], inv_freq [d / 2]
// on the GPU, query [b, hq, n, d] or None (of one layer), stream) -> the rotated query, or True; None if not taken.
PyObject* rope_rows(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  c10::Device dev(c10::DeviceType::CPU);
  if (n_args != 8 || !current(a[4], &dev)) Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i)
    if (!PyList_CheckExact(a[i]) && !PyTuple_CheckExact(a[i])) Py_RETURN_NONE;
  const Py_ssize_t layers = PySequence_Fast_GET_SIZE(a[0]);
  if (layers < 1) Py_RETURN_NONE;
  for (int i = 1; i < 4; ++i)
    if (PySequence_Fast_GET_SIZE(a[i]) != layers) Py_RETURN_NONE;
  const at::Tensor *slots = tensor(a[4], dev), *freq = tensor(a[5], dev), *pool = tensor(PySequence_Fast_GET_ITEM(a[2], 0), dev);
  if (!slots || !freq || !pool || slots->dim() != 3 || slots->size(2) != 4 || !table(*slots)) Py_RETURN_NONE;
  if (freq->scalar_type() != at::kFloat || freq->dim() != 1 || freq->size(0) != kHeadDim / 2 || !freq->is_contiguous()) Py_RETURN_NONE;
  int dt;
  if (pool->dim() != 4 || pool->size(3) != kHeadDim || pool->stride(3) != 1 || !dtype_code(*pool, &dt)) Py_RETURN_NONE;
  const int64_t b = slots->size(0), n = slots->size(1);
  int64_t sk[3], sv[3], sq[3] = {0, 0, 0}, so[3] = {0, 0, 0}, hk = 0, hv = 0, hq = 0;
  std::vector<const void*> ks, vs;
  std::vector<void*> kps, vps;
  if (!row_list(a[0], dev, pool->scalar_type(), b, n, &hk, &ks, sk) ||
      !row_list(a[1], dev, pool->scalar_type(), b, n, &hv, &vs, sv) || hk != pool->size(1) || hv != hk ||
      !pool_list(a[2], dev, *pool, &kps) || !pool_list(a[3], dev, *pool, &vps) || watched())
    Py_RETURN_NONE;
  at::Tensor out;
  const void* qp = nullptr;
  void* op = nullptr;
  if (a[6] != Py_None) {
    const at::Tensor* q = tensor(a[6], dev);
    if (!q || layers != 1 || !same_type(*pool, *q) || q->dim() != 4 || q->size(0) != b || q->size(2) != n ||
        q->size(3) != kHeadDim || q->stride(3) != 1 || recorded(*q))
      Py_RETURN_NONE;
    hq = q->size(1);
    if (hq < 1) Py_RETURN_NONE;
    out = at::empty({b, hq, n, kHeadDim}, q->options().requires_grad(false));
    for (int i = 0; i < 3; ++i) {
      sq[i] = stride(*q, i);
      so[i] = stride(out, i);
    }
    qp = q->const_data_ptr();
    op = out.mutable_data_ptr();
  }
  void* stream = raw_stream(a[7]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t sp[3] = {pool->stride(0), pool->stride(1), pool->stride(2)};
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = tc_paged_append_rope(ks.data(), sk, vs.data(), sv, kps.data(), vps.data(), sp, static_cast<int>(pool->size(0)),
                            static_cast<int>(pool->size(2)), words(*slots), &qp, sq, &op, so, static_cast<int>(hq),
                            nullptr, static_cast<const float*>(freq->const_data_ptr()), static_cast<int>(layers),
                            static_cast<int>(b), static_cast<int>(hk), n, kHeadDim, dt, stream);
  Py_END_ALLOW_THREADS
  if (rc != TC_OK) Py_RETURN_NONE;
  for (int i = 2; i < 4; ++i)
    for (Py_ssize_t l = 0; l < layers; ++l) {
      const at::Tensor& t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(a[i], l));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
  if (hq) return THPVariable_Wrap(std::move(out));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}

}  // namespace

PyMODINIT_FUNC PyInit__fast() {
  static PyMethodDef methods[] = {
      {"decode", fast(decode), METH_FASTCALL, "decode(query, key, value, scale, stream[, window, sinks]) -> out or None"},
      {"decode_append", fast(decode_append), METH_FASTCALL,
       "decode_append(query, k_buf, v_buf, k_new, v_new, n_or_pos, scale, stream[, window, sinks]) -> out or None"},
      {"decode_shared", fast(decode_shared), METH_FASTCALL,
       "decode_shared(q, k_prefix, v_prefix, k, v, lens, out, scale, stream) -> out or None"},
      {"paged_decode", fast(paged_decode), METH_FASTCALL,
       "paged_decode(q, k_pool, v_pool, table, counts, out, scale, stream) -> out or None"},
      {"paged_shared", fast(paged_shared), METH_FASTCALL,
       "paged_shared(q, k_pool, v_pool, shared, table, counts, k_new, v_new, out, scale, stream) -> out or None"},
      {"rope_rows", fast(rope_rows), METH_FASTCALL,
       "rope_rows(ks, vs, k_pools, v_pools, slots, inv_freq, query, stream) -> rotated query, True or None"},
      {"paged_append", fast(paged_append), METH_FASTCALL,
       "paged_append(q, k_pool, v_pool, table, counts, k_new, v_new, out, scale, stream) -> out or None"},
      {"append_rows", fast(append_rows), METH_FASTCALL, "append_rows(k_buf, v_buf, row0, k, v, stream) -> bool"},
      {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "Native call paths of the wrappers.", -1, methods};
  PyObject* m = PyModule_Create(&module);
  // The torch whose headers these paths were compiled with: they read its tensors in place, so they serve no other.
  if (m && PyModule_AddStringConstant(m, "torch_version", TC_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}
