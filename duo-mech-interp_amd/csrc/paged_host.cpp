// The host side of the paged-cache ops as a Python extension: the checks of their arguments, their outputs and workspaces, and
// the call of the C ABI, whose functions bind() receives as addresses (the library stays the one that the ctypes binding
// loaded). A decode step makes these calls eagerly for every layer, and from Python the checks, two allocations and a
// conversion of up to 45 arguments took longer than the kernels: append 10.9 us a call against 4.3 here, read-back 11.1 and
// 6.0, attention 17.3 and 8.6 (two launches of 2.8), verification 14.2 and 8.9.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <string>

#include "q35hip.h"

namespace {

using at::Tensor;

struct Refused {
  std::string msg;
};
[[noreturn]] void refuse(const std::string& msg) { throw Refused{"q35hip: " + msg}; }
constexpr const char* kNotOnGpu = "inputs must be HIP device tensors (there is no CPU fallback)";

PyObject* g_error = nullptr;   // the exception that refusals raise
PyObject* g_check = nullptr;   // check(status, name): raises for a status that is not 0
PyObject* g_stream = nullptr;  // the current stream's handle of a device
decltype(&q35_paged_kv_append) g_append = nullptr;
decltype(&q35_paged_kv_rows) g_rows = nullptr;
decltype(&q35_gated_attn_paged_workspace_bytes) g_attn_bytes = nullptr;
decltype(&q35_gated_attn_paged) g_attn = nullptr;
decltype(&q35_verify_drafts_workspace_bytes) g_verify_bytes = nullptr;
decltype(&q35_verify_drafts) g_verify = nullptr;
decltype(&q35_gated_attn_paged_shared_workspace_bytes) g_shared_bytes = nullptr;
decltype(&q35_gated_attn_paged_shared) g_shared = nullptr;
decltype(&q35_sample_tokens_workspace_bytes) g_sample_bytes = nullptr;
decltype(&q35_sample_tokens) g_sample = nullptr;
decltype(&q35_quantize_rows_i8) g_quantize = nullptr;
decltype(&q35_add_rmsnorm_i8) g_norm_i8 = nullptr;
decltype(&q35_gemm_i8) g_gemm_i8 = nullptr;

// A Python error is set already.
struct PyFailed {};

const Tensor* optional(PyObject* o) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("inputs must be tensors");
  return &THPVariable_Unpack(o);
}
const Tensor& tensor(PyObject* o) {
  const Tensor* t = optional(o);
  if (!t) refuse("inputs must be tensors");
  return *t;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailed{};
  return v;
}
// A device tensor whose memory holds its values, as nobody else's business: not a functorch or functionalization wrapper, a
// subclass, a view that is negated or conjugated when read, and nothing that autograd follows.
bool plain(PyObject* o) {
  if (!THPVariable_Check(o)) return true;  // (a number or None)
  if (!THPVariable_CheckExact(o)) return false;
  constexpr c10::DispatchKeySet own({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradCUDA,
                                     c10::DispatchKey::AutocastCUDA});
  const Tensor& t = THPVariable_Unpack(o);
  return (t.key_set().raw_repr() & ~own.raw_repr()) == 0 && !(at::GradMode::is_enabled() && t.requires_grad());
}

template <typename T = void> T* data(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T = void> T* data(const Tensor* t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

bool is(const Tensor& t, at::ScalarType s) { return t.scalar_type() == s; }
bool dense_on(int64_t d, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) {
    if (!t) continue;
    if (!t->is_cuda()) refuse(kNotOnGpu);
    if (t->get_device() != d || !t->is_contiguous()) return false;
  }
  return true;
}
bool ints_per_row(const Tensor* t, int64_t B) { return !t || (is(*t, at::kInt) && t->dim() == 1 && t->size(0) == B); }

// A [B, T, H, 256] fp32 or bf16 view: rows of 256 dense, anything else strided.
struct View {
  int64_t b, t, h;
  int dtype;
};
View heads_view(const Tensor& x, const char* what) {
  if (!x.is_cuda()) refuse(kNotOnGpu);
  if (x.dim() != 4 || x.stride(3) != 1 || x.size(3) != 256 || !(is(x, at::kFloat) || is(x, at::kBFloat16)))
    refuse(std::string(what) + ": [B, T, heads, 256] fp32 or bf16 with dense rows");
  return {x.stride(0), x.stride(1), x.stride(2), is(x, at::kFloat) ? Q35_F32 : Q35_BF16};
}

struct Pages {
  const Tensor &k, &v;
  const Tensor *ks, *vs;
  const Tensor &table, &pos;
  const Tensor* lens;
  int fmt;
  int64_t n, heads, size, blocks, ld;
};
// k_pages, v_pages, k_scale, v_scale, table, pos, lens, checked for B rows (B < 0: as many as the table has) on device d
// (d < 0: the pages' own).
Pages pages_of(PyObject* const* a, int64_t d, int64_t B) {
  Pages p{tensor(a[0]), tensor(a[1]), optional(a[2]), optional(a[3]), tensor(a[4]), tensor(a[5]), optional(a[6]),
          0,            0,            0,              0,              0,            0};
  if (!p.k.is_cuda()) refuse(kNotOnGpu);
  if (d < 0) d = p.k.get_device();
  if (!dense_on(d, {&p.k, &p.v, p.ks, p.vs, &p.pos, p.lens}))
    refuse("pages, pos and lens must be contiguous and on one device with the other inputs");
  if (!p.table.is_cuda()) refuse(kNotOnGpu);
  if (p.table.dim() != 2 || !is(p.table, at::kInt) || p.table.get_device() != d || p.table.stride(1) != 1 ||
      (B >= 0 && p.table.size(0) != B))
    refuse("table: [B, blocks] int32 with dense rows, on the pages' device");
  p.blocks = p.table.size(1);
  p.ld = p.table.stride(0);
  B = p.table.size(0);
  if (!ints_per_row(&p.pos, B) || !ints_per_row(p.lens, B)) refuse("pos, lens: [B] int32");
  if (p.k.dim() != 4 || p.v.sizes() != p.k.sizes() || p.v.scalar_type() != p.k.scalar_type())
    refuse("pages: k and v alike, [pages, Hkv, page size, ...]");
  p.n = p.k.size(0), p.heads = p.k.size(1), p.size = p.k.size(2);
  if (is(p.k, at::kBFloat16)) {
    if (p.k.size(3) != 256) refuse("bf16 pages: [pages, Hkv, page size, 256]");
    p.fmt = Q35_BF16;
    return p;
  }
  if (!is(p.k, at::kByte) || p.k.size(3) != 128) refuse("4-bit pages: [pages, Hkv, page size, 128] uint8");
  for (const Tensor* s : {p.ks, p.vs})
    if (!s || !is(*s, at::kBFloat16) || s->dim() != 4 || s->size(0) != p.n || s->size(1) != p.heads || s->size(2) != p.size ||
        s->size(3) != 4)
      refuse("4-bit pages: k_scale, v_scale [pages, Hkv, page size, 4] bf16");
  p.fmt = Q35_I4_G64;
  return p;
}

// Their addresses.
struct PagesAt {
  void *k, *v, *ks, *vs;
  int32_t *table, *pos, *lens;
  explicit PagesAt(const Pages& p)
      : k(data(p.k)), v(data(p.v)), ks(data(p.ks)), vs(data(p.vs)), table(data<int32_t>(p.table)), pos(data<int32_t>(p.pos)),
        lens(data<int32_t>(p.lens)) {}
};

struct Rope {
  const Tensor &cos, &sin;
  const Tensor* norm_w;
  int64_t rot;
};
// cos, sin, norm_w, with tables of at least `rows` positions.
Rope rope_of(PyObject* const* a, int64_t d, int64_t rows) {
  Rope r{tensor(a[0]), tensor(a[1]), optional(a[2]), 0};
  if (!dense_on(d, {&r.cos, &r.sin, r.norm_w}))
    refuse("cos, sin and the norm weight must be contiguous and on one device with the other inputs");
  if (!is(r.cos, at::kFloat) || !is(r.sin, at::kFloat) || r.cos.dim() != 2 || r.sin.sizes() != r.cos.sizes() ||
      (r.norm_w && (!is(*r.norm_w, at::kFloat) || r.norm_w->dim() != 1 || r.norm_w->size(0) != 256)))
    refuse("cos, sin: [P, rot / 2] fp32; norm weight: [256] fp32");
  if (r.cos.size(0) < rows && r.cos.size(1)) refuse("cos/sin tables need " + std::to_string(rows) + " rows");
  r.rot = 2 * r.cos.size(1);
  return r;
}

struct RopeAt {
  float *cos, *sin, *norm_w;
  explicit RopeAt(const Rope& r) : cos(data<float>(r.cos)), sin(data<float>(r.sin)), norm_w(data<float>(r.norm_w)) {}
};

// An empty tensor next to `like`, from the allocator that like's memory came from (the caching one; a dispatch of at::empty takes
// half a microsecond more, and a call makes up to three).
Tensor make(at::IntArrayRef size, at::ScalarType s, const Tensor& like) {
  c10::Allocator* from = like.has_storage() ? like.storage().allocator() : nullptr;
  if (!from) return at::empty(size, at::TensorOptions().dtype(s).device(like.device()));
  const c10::DeviceGuard guard(like.device());
  return Tensor(at::detail::empty_generic(size, from, c10::DispatchKeySet(c10::DispatchKey::CUDA), s, std::nullopt));
}

// Gives the interpreter lock up for as long as it lives, however its scope is left.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// call(stream) with t's device current and the interpreter free, its status checked. `call` holds its pointers already (init
// captures of the lambda): a tensor without storage refuses to give one, by an exception, and before anything runs.
template <typename F> void launch(const Tensor& t, const char* name, F&& call) {
  PyObject* d = PyLong_FromLongLong(t.get_device());
  PyObject* h = d ? PyObject_CallOneArg(g_stream, d) : nullptr;
  Py_XDECREF(d);
  if (!h) throw PyFailed{};
  void* stream = PyLong_AsVoidPtr(h);
  Py_DECREF(h);
  if (PyErr_Occurred()) throw PyFailed{};
  int status;
  {
    const c10::DeviceGuard guard(t.device());
    const Unlocked unlocked;
    status = call(static_cast<q35_stream_t>(stream));
  }
  if (status != Q35_OK) {
    Py_XDECREF(PyObject_CallFunction(g_check, "is", status, name));
    if (!PyErr_Occurred()) refuse(name);
    throw PyFailed{};
  }
}

// f(arguments) for exactly n of them, with every C++ exception as a Python one.
template <typename F> PyObject* guarded(Py_ssize_t n, Py_ssize_t want, F&& f) {
  try {
    if (!g_error) {
      PyErr_SetString(PyExc_RuntimeError, "q35hip: the host module is not bound");
      return nullptr;
    }
    if (n != want) refuse("wrong number of arguments");
    return f();
  } catch (const PyFailed&) {
  } catch (const Refused& r) {
    PyErr_SetString(g_error, r.msg.c_str());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// k, v, k_pages, v_pages, k_scale, v_scale, table, pos, lens, cos, sin, k_norm_w, eps
PyObject* paged_kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const Tensor &k = tensor(a[0]), &v = tensor(a[1]);
    const View kv = heads_view(k, "k"), vv = heads_view(v, "v");
    const int64_t B = k.size(0), T = k.size(1), d = k.get_device();
    const Pages p = pages_of(a + 2, d, B);
    if (v.sizes() != k.sizes() || vv.dtype != kv.dtype || v.get_device() != d || p.heads != k.size(2))
      refuse("k, v: alike, with the pages' heads");
    const Rope r = rope_of(a + 9, d, p.blocks * p.size);
    const double eps = number(a[12]);
    if (B && T)
      launch(k, "q35_paged_kv_append", [&, at = PagesAt(p), ro = RopeAt(r), xk = data(k), xv = data(v)](q35_stream_t st) {
        return g_append(xk, kv.b, kv.t, kv.h, xv, vv.b, vv.t, vv.h, kv.dtype, ro.norm_w, (float)eps, ro.cos, ro.sin, r.rot,
                        at.table, p.ld, p.blocks, at.pos, at.lens, at.k, at.v, at.ks, at.vs, p.fmt, p.n, p.size, B, T,
                        p.heads, 256, st);
      });
    Py_RETURN_NONE;
  });
}

// k_pages, v_pages, k_scale, v_scale, table, pos, lens, T -> (k, v)
PyObject* paged_kv_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Pages p = pages_of(a, -1, -1);
    const int64_t T = integer(a[7]), B = p.table.size(0);
    if (T < 0) refuse("T: a number of tokens");
    const Tensor k = make({B, p.heads, T, 256}, at::kBFloat16, p.k), v = make({B, p.heads, T, 256}, at::kBFloat16, p.k);
    if (B && T)
      launch(p.k, "q35_paged_kv_rows", [&, at = PagesAt(p), ko = data(k), vo = data(v)](q35_stream_t st) {
        return g_rows(at.k, at.v, at.ks, at.vs, p.fmt, p.n, p.size, at.table, p.ld, p.blocks, at.pos, at.lens, ko, vo, B, T,
                      p.heads, 256, st);
      });
    return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  });
}

// q, gate, k_pages, v_pages, k_scale, v_scale, table, pos, lens, cos, sin, q_norm_w, eps, scale, splits, f32_out -> out
PyObject* gated_attn_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const Tensor& q = tensor(a[0]);
    const Tensor* gate = optional(a[1]);
    const View qv = heads_view(q, "q");
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), d = q.get_device();
    const Pages p = pages_of(a + 2, d, B);
    View gv{0, 0, 0, qv.dtype};
    if (gate) {
      gv = heads_view(*gate, "gate");
      if (gate->sizes() != q.sizes() || gv.dtype != qv.dtype || gate->get_device() != d) refuse("gate: like q");
    }
    const Rope r = rope_of(a + 9, d, p.blocks * p.size);
    const double eps = number(a[12]), scale = number(a[13]);
    const int64_t splits = integer(a[14]);
    const int f32 = PyObject_IsTrue(a[15]);
    if (f32 < 0) throw PyFailed{};
    const Tensor out = make({B, T, Hq * 256}, f32 ? at::kFloat : at::kBFloat16, q);
    if (out.numel()) {
      const size_t bytes = g_attn_bytes(B, T, Hq, p.heads, 256, p.blocks, p.size, splits);
      if (!bytes) refuse("unsupported attention shape");
      const Tensor ws = make({(int64_t)bytes}, at::kByte, q);
      launch(q, "q35_gated_attn_paged", [&, at = PagesAt(p), ro = RopeAt(r), xq = data(q), xg = data(gate), o = data(out),
                                         w = data(ws)](q35_stream_t st) {
        return g_attn(xq, qv.b, qv.t, qv.h, xg, gv.b, gv.t, gv.h, qv.dtype, ro.norm_w, (float)eps, ro.cos, ro.sin, r.rot,
                      at.k, at.v, at.ks, at.vs, p.fmt, p.n, p.size, at.table, p.ld, p.blocks, at.pos, at.lens, o,
                      f32 ? Q35_F32 : Q35_BF16, B, T, Hq, p.heads, 256, (float)scale, splits, w, bytes, st);
      });
    }
    return THPVariable_Wrap(out);
  });
}

// logits, draft_ids, draft_probs, u, lens, temperatures, temperature -> (n_accept, tokens)
PyObject* verify_drafts(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &ids = tensor(a[1]), &u = tensor(a[3]);
    const Tensor *probs = optional(a[2]), *lens = optional(a[4]), *temps = optional(a[5]);
    const double temperature = number(a[6]);
    if (!x.is_cuda() || !ids.is_cuda() || !u.is_cuda() || (probs && !probs->is_cuda())) refuse(kNotOnGpu);
    const int64_t d = x.get_device();
    if (!dense_on(d, {lens, temps}) || ids.get_device() != d || u.get_device() != d || (probs && probs->get_device() != d))
      refuse("inputs must be on one device, lens and temperature contiguous");
    if (x.dim() != 3 || !is(x, at::kFloat) || x.stride(2) != 1 || x.size(1) == 0)
      refuse("logits: [B, K + 1, V] fp32 with dense rows");
    const int64_t B = x.size(0), K = x.size(1) - 1, V = x.size(2);
    if (ids.dim() != 2 || ids.size(0) != B || ids.size(1) != K || !is(ids, at::kInt) || (K > 1 && ids.stride(1) != 1))
      refuse("draft_ids: [B, K] int32 with dense rows");
    if (u.dim() != 2 || u.size(0) != B || u.size(1) != K + 1 || !is(u, at::kFloat) || (K && u.stride(1) != 1))
      refuse("u: [B, K + 1] fp32 with dense rows");
    if (probs && (probs->dim() != 3 || probs->size(0) != B || probs->size(1) != K || probs->size(2) != V ||
                  !is(*probs, at::kFloat) || probs->stride(2) != 1))
      refuse("draft_probs: [B, K, V] fp32 with dense rows");
    if (!ints_per_row(lens, B) || (temps && (!is(*temps, at::kFloat) || temps->dim() != 1 || temps->size(0) != B)))
      refuse("lens: [B] int32; temperature: a number of at least 0 or [B] fp32");
    const Tensor accepted = make({B}, at::kInt, x), tokens = make({B, K + 1}, at::kInt, x);
    if (B) {
      const size_t bytes = g_verify_bytes(B, K, V);
      if (!bytes)
        refuse("unsupported draft shape (B=" + std::to_string(B) + ", K=" + std::to_string(K) + ", V=" + std::to_string(V) +
               ")");
      const Tensor ws = make({(int64_t)bytes}, at::kByte, x);
      const int64_t xs[2] = {x.stride(0), x.stride(1)}, qs[2] = {probs ? probs->stride(0) : 0, probs ? probs->stride(1) : 0};
      const int64_t is = ids.stride(0), us = u.stride(0);
      launch(x, "q35_verify_drafts", [&, xa = data<float>(x), ia = data<int32_t>(ids), qa = data<float>(probs),
                                      ua = data<float>(u), la = data<int32_t>(lens), ta = data<float>(temps),
                                      na = data<int32_t>(accepted), ka = data<int32_t>(tokens), w = data(ws)](q35_stream_t st) {
        return g_verify(xa, xs[0], xs[1], ia, is, qa, qs[0], qs[1], ua, us, la, ta, (float)temperature, na, ka, B, K, V, w,
                        bytes, st);
      });
    }
    return Py_BuildValue("(NN)", THPVariable_Wrap(accepted), THPVariable_Wrap(tokens));
  });
}

// As gated_attn_paged up to scale, then f32_out, shared_blocks -> out
PyObject* gated_attn_paged_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 16, [&]() -> PyObject* {
    const Tensor& q = tensor(a[0]);
    const Tensor* gate = optional(a[1]);
    const View qv = heads_view(q, "q");
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), d = q.get_device();
    const Pages p = pages_of(a + 2, d, B);
    View gv{0, 0, 0, qv.dtype};
    if (gate) {
      gv = heads_view(*gate, "gate");
      if (gate->sizes() != q.sizes() || gv.dtype != qv.dtype || gate->get_device() != d) refuse("gate: like q");
    }
    const Rope r = rope_of(a + 9, d, p.blocks * p.size);
    const double eps = number(a[12]), scale = number(a[13]);
    const int f32 = PyObject_IsTrue(a[14]);
    if (f32 < 0) throw PyFailed{};
    const int64_t shared = integer(a[15]);
    if (shared < 0 || shared > p.blocks) refuse("shared_blocks: 0 up to the table's blocks");
    const Tensor out = make({B, T, Hq * 256}, f32 ? at::kFloat : at::kBFloat16, q);
    if (out.numel()) {
      const size_t bytes = g_shared_bytes(B, T, Hq, p.heads, 256, p.blocks, p.size, shared);
      if (!bytes) refuse("unsupported attention shape");
      const Tensor ws = make({(int64_t)bytes}, at::kByte, q);
      launch(q, "q35_gated_attn_paged_shared", [&, at = PagesAt(p), ro = RopeAt(r), xq = data(q), xg = data(gate), o = data(out),
                                                w = data(ws)](q35_stream_t st) {
        return g_shared(xq, qv.b, qv.t, qv.h, xg, gv.b, gv.t, gv.h, qv.dtype, ro.norm_w, (float)eps, ro.cos, ro.sin, r.rot,
                        at.k, at.v, at.ks, at.vs, p.fmt, p.n, p.size, at.table, p.ld, p.blocks, shared, at.pos, at.lens, o,
                        f32 ? Q35_F32 : Q35_BF16, B, T, Hq, p.heads, 256, (float)scale, w, bytes, st);
      });
    }
    return THPVariable_Wrap(out);
  });
}

// temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p: a row's settings
struct Cuts {
  const Tensor *t, *k, *p, *m;
  double temperature, top_p, min_p;
  int64_t top_k;
};
Cuts cuts_of(PyObject* const* a, int64_t d, int64_t B) {
  const Cuts c{optional(a[0]), optional(a[2]), optional(a[4]), optional(a[6]),
               number(a[1]),   number(a[5]),   number(a[7]),   integer(a[3])};
  if (!dense_on(d, {c.t, c.k, c.p, c.m})) refuse("per-row settings must be contiguous and on the logits' device");
  for (const Tensor* s : {c.t, c.p, c.m})
    if (s && (!is(*s, at::kFloat) || s->dim() != 1 || s->size(0) != B))
      refuse("temperature, top_p, min_p: numbers or [B] fp32");
  if (!ints_per_row(c.k, B)) refuse("top_k: a number or [B] int32");
  if (!(c.temperature >= 0) || c.top_p != c.top_p || c.min_p != c.min_p)
    refuse("temperature: at least 0; top_p, min_p: numbers");
  return c;
}
// Logits [B, V] or [B, P, V] with dense rows.
struct Logits {
  int64_t B, P, V, sb, sp;
};
Logits logits_of(const Tensor& x, bool positions) {
  if (!x.is_cuda()) refuse(kNotOnGpu);
  const bool three = x.dim() == 3;
  if (!(x.dim() == 2 || (positions && three)) || !is(x, at::kFloat) || x.stride(-1) != 1 || x.size(-1) == 0)
    refuse(positions ? "logits: [B, V] or [B, P, V] fp32 with dense rows" : "logits: [B, V] fp32 with dense rows");
  return {x.size(0), three ? x.size(1) : 1, x.size(-1), x.stride(0), three ? x.stride(1) : x.size(-1)};
}
void sample(const Tensor& x, const Logits& l, const Tensor* u, const Cuts& c, const Tensor* tokens, int kind, const Tensor* out) {
  const size_t bytes = g_sample_bytes(l.B, l.P, l.V);
  if (!bytes) refuse("unsupported number of rows or tokens");
  const Tensor ws = make({(int64_t)bytes}, at::kByte, x);
  const int64_t us = u ? u->stride(0) : 0;
  launch(x, "q35_sample_tokens", [&, xa = data<float>(x), ua = data<float>(u), ta = data<float>(c.t), ka = data<int32_t>(c.k),
                                  pa = data<float>(c.p), ma = data<float>(c.m), to = data<int32_t>(tokens), o = data<float>(out),
                                  w = data(ws)](q35_stream_t st) {
    return g_sample(xa, l.sb, l.sp, ua, us, ta, (float)c.temperature, ka, c.top_k, pa, (float)c.top_p, ma, (float)c.min_p, to,
                    kind, o, l.B, l.P, l.V, w, bytes, st);
  });
}

// logits, u, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p, want_probs -> (tokens, probs), or tokens
PyObject* sample_tokens(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &u = tensor(a[1]);
    const Logits l = logits_of(x, false);
    const int64_t d = x.get_device();
    if (!u.is_cuda()) refuse(kNotOnGpu);
    if (u.get_device() != d || !is(u, at::kFloat) || u.dim() != 1 || u.size(0) != l.B)
      refuse("u: [B] fp32 on the logits' device");
    const Cuts c = cuts_of(a + 2, d, l.B);
    const int want = PyObject_IsTrue(a[10]);
    if (want < 0) throw PyFailed{};
    const Tensor tokens = make({l.B}, at::kInt, x), probs = want ? make({l.B, l.V}, at::kFloat, x) : Tensor();
    if (l.B) sample(x, l, &u, c, &tokens, want, want ? &probs : nullptr);
    if (!want) return THPVariable_Wrap(tokens);
    return Py_BuildValue("(NN)", THPVariable_Wrap(tokens), THPVariable_Wrap(probs));
  });
}

// logits, temperatures, temperature, top_ks, top_k, top_ps, top_p, min_ps, min_p -> logits
PyObject* filter_logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Tensor& x = tensor(a[0]);
    const Logits l = logits_of(x, true);
    const Cuts c = cuts_of(a + 1, x.get_device(), l.B);
    const Tensor out = make(x.sizes(), at::kFloat, x);
    if (l.B && l.P) sample(x, l, nullptr, c, nullptr, 2, &out);
    return THPVariable_Wrap(out);
  });
}

// Rows [..., K] whose last dim is dense and that are evenly strided: how many, and how far apart.
struct Rows {
  int64_t M, K, ld;
};
Rows rows_of(const Tensor& x, const char* what) {
  if (x.dim() < 1 || x.size(-1) == 0 || x.stride(-1) != 1) refuse(std::string(what) + ": [..., K] with dense rows");
  const int64_t K = x.size(-1), M = x.numel() / K;
  int64_t ld = K;
  if (x.dim() > 1 && M > 1) {
    int64_t at = x.dim() - 2;
    while (at > 0 && x.size(at) == 1) --at;
    ld = x.stride(at);
    int64_t want = ld * x.size(at);
    for (int64_t i = at - 1; i >= 0; --i) {
      if (x.size(i) != 1 && x.stride(i) != want) refuse(std::string(what) + ": rows must be evenly strided");
      want *= x.size(i);
    }
    if (ld < K) refuse(std::string(what) + ": rows must not overlap");
  }
  return {M, K, ld};
}
Tensor scales_for(const Tensor& x) {
  return make(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
}

// x -> (q, s)
PyObject* quantize_rows_i8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    const Tensor& x = tensor(a[0]);
    if (!x.is_cuda()) refuse(kNotOnGpu);
    if (!(is(x, at::kFloat) || is(x, at::kBFloat16))) refuse("x: fp32 or bf16");
    const Rows r = rows_of(x, "x");
    const Tensor q = make(x.sizes(), at::kChar, x), s = scales_for(x);
    if (r.M)
      launch(x, "q35_quantize_rows_i8", [&, xa = data(x), qa = data<int8_t>(q), sa = data<float>(s)](q35_stream_t st) {
        return g_quantize(xa, r.ld, is(x, at::kFloat) ? Q35_F32 : Q35_BF16, qa, sa, r.M, r.K, st);
      });
    return Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(s));
  });
}

// x, y, w, eps -> (q, s); x += y in place
PyObject* add_rmsnorm_i8_(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const Tensor &x = tensor(a[0]), &w = tensor(a[2]);
    const Tensor* y = optional(a[1]);
    const double eps = number(a[3]);
    if (!x.is_cuda() || !w.is_cuda() || (y && !y->is_cuda())) refuse(kNotOnGpu);
    const int64_t d = x.get_device();
    if (!is(x, at::kFloat) || (y && (!is(*y, at::kFloat) || y->sizes() != x.sizes() || y->get_device() != d)))
      refuse("x: fp32; y like x");
    const Rows r = rows_of(x, "x"), ry = y ? rows_of(*y, "y") : Rows{0, 0, 0};
    if (!dense_on(d, {&w}) || !is(w, at::kFloat) || w.numel() != r.K) refuse("w: [K] fp32 on x's device");
    const Tensor q = make(x.sizes(), at::kChar, x), s = scales_for(x);
    if (r.M)
      launch(x, "q35_add_rmsnorm_i8", [&, xa = data<float>(x), ya = data<float>(y), wa = data<float>(w), qa = data<int8_t>(q),
                                       sa = data<float>(s)](q35_stream_t st) {
        return g_norm_i8(xa, r.ld, ya, ry.ld, wa, qa, sa, r.M, r.K, (float)eps, st);
      });
    return Py_BuildValue("(NN)", THPVariable_Wrap(q), THPVariable_Wrap(s));
  });
}

// q, q_scale, W, w_scale, y or None, epilogue, pushes, T, cap -> y
PyObject* gemm_i8_(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const Tensor &q = tensor(a[0]), &qs = tensor(a[1]), &W = tensor(a[2]), &ws = tensor(a[3]);
    const Tensor *given = optional(a[4]), *pushes = optional(a[6]), *cap = optional(a[8]);
    const int64_t epilogue = integer(a[5]), T = integer(a[7]);
    if (!q.is_cuda() || !W.is_cuda() || (given && !given->is_cuda())) refuse(kNotOnGpu);
    const int64_t d = q.get_device();
    if (!dense_on(d, {&qs, &W, &ws, pushes})) refuse("scales, W and pushes must be contiguous and on q's device");
    if (!is(q, at::kChar) || !is(W, at::kChar) || W.dim() != 2 || !is(qs, at::kFloat) || !is(ws, at::kFloat))
      refuse("q: [..., K] int8, W: [N, K] int8, scales fp32");
    const Rows r = rows_of(q, "q");
    const int64_t N = W.size(0), M = r.M;
    if (W.size(1) != r.K || qs.numel() != M || ws.dim() != 1 || ws.size(0) != N)
      refuse("q, W and their scales disagree (q_scale: one a row of q, w_scale: [N])");
    const bool swiglu = epilogue == 2;
    const int64_t No = swiglu ? N / 2 : N;
    if (swiglu && N % 2) refuse("SwiGLU: W holds (gate, up) pairs of rows");
    Tensor y;
    if (given) {
      y = *given;
    } else {
      auto sz = q.sizes().vec();
      sz.back() = No;
      y = make(sz, at::kFloat, q);
    }
    if (!is(y, at::kFloat) || y.get_device() != d || y.dim() < 1 || y.size(-1) != No || y.numel() != M * No)
      refuse("y: one row of N (SwiGLU: N / 2) fp32 for each of q's, on its device");
    if (pushes && (!is(*pushes, at::kInt) || pushes->dim() != 2 || pushes->size(1) != 6))
      refuse("pushes: [n, 6] int32 records (see pack_pushes)");
    int64_t ldc = 0, ldcr = 0;
    if (cap) {
      if (!swiglu || !cap->is_cuda() || cap->get_device() != d || !is(*cap, at::kFloat) || cap->dim() < 2 ||
          cap->dim() > 3 || cap->stride(-1) != 1 || cap->size(-1) != No || cap->numel() != M * No || T < 1 ||
          (cap->dim() == 3 && cap->size(1) != T))
        refuse("capture (SwiGLU only): [rows, T, N / 2] or [M, N / 2] fp32 on q's device with unit neuron stride");
      ldc = cap->stride(-2);
      ldcr = cap->dim() == 3 ? cap->stride(0) : ldc * T;
    }
    if (M && No) {
      const Rows ry = rows_of(y, "y");
      launch(q, "q35_gemm_i8", [&, qa = data<int8_t>(q), sa = data<float>(qs), wa = data<int8_t>(W), wsa = data<float>(ws),
                                ya = data<float>(y), pa = static_cast<const q35_push*>(data(pushes)),
                                ca = data<float>(cap)](q35_stream_t st) {
        return g_gemm_i8(qa, M > 1 ? r.ld : r.K, sa, wa, wsa, ya, ry.ld, M, N, r.K, (int)epilogue, pa,
                         pushes ? pushes->size(0) : 0, T, ca, ldc, ldcr, st);
      });
    }
    return THPVariable_Wrap(y);
  });
}

// Whether an op on these arguments is the functions above and nothing more. Whatever follows a thread's calls (a trace, a
// dispatch mode, a transform) has its key among those that the thread includes in every dispatch.
bool direct_on(PyObject* const* a, Py_ssize_t n) {
  constexpr c10::DispatchKeySet always({c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView});
  const auto local = c10::impl::tls_local_dispatch_key_set();
  const bool followed = (local.included_.raw_repr() & ~local.excluded_.raw_repr() & ~always.raw_repr()) != 0;
  return !followed && std::all_of(a, a + n, plain);
}
// Any arguments -> that as a bool.
PyObject* direct(PyObject*, PyObject* const* a, Py_ssize_t n) { return PyBool_FromLong(direct_on(a, n)); }
// The op where it is so, else NotImplemented.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* try_direct(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  if (direct_on(a, n)) return F(self, a, n);
  Py_RETURN_NOTIMPLEMENTED;
}

// error, check, stream, then the addresses of the six functions of the C ABI
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "bind: error, check, stream and six addresses");
    return nullptr;
  }
  void* f[6];
  for (int i = 0; i < 6; ++i) {
    f[i] = PyLong_AsVoidPtr(a[3 + i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_rows = reinterpret_cast<decltype(g_rows)>(f[1]);
  g_attn_bytes = reinterpret_cast<decltype(g_attn_bytes)>(f[2]);
  g_attn = reinterpret_cast<decltype(g_attn)>(f[3]);
  g_verify_bytes = reinterpret_cast<decltype(g_verify_bytes)>(f[4]);
  g_verify = reinterpret_cast<decltype(g_verify)>(f[5]);
  PyObject** to[3] = {&g_error, &g_check, &g_stream};
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(a[i]);
    Py_XDECREF(*to[i]);
    *to[i] = a[i];
  }
  Py_RETURN_NONE;
}

// the addresses of the seven functions of the C ABI that came later
PyObject* bind_sampling(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "bind_sampling: seven addresses");
    return nullptr;
  }
  void* f[7];
  for (int i = 0; i < 7; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_shared_bytes = reinterpret_cast<decltype(g_shared_bytes)>(f[0]);
  g_shared = reinterpret_cast<decltype(g_shared)>(f[1]);
  g_sample_bytes = reinterpret_cast<decltype(g_sample_bytes)>(f[2]);
  g_sample = reinterpret_cast<decltype(g_sample)>(f[3]);
  g_quantize = reinterpret_cast<decltype(g_quantize)>(f[4]);
  g_norm_i8 = reinterpret_cast<decltype(g_norm_i8)>(f[5]);
  g_gemm_i8 = reinterpret_cast<decltype(g_gemm_i8)>(f[6]);
  Py_RETURN_NONE;
}

#define Q35_FAST(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
#define Q35_METHOD(f) Q35_FAST(#f, f), Q35_FAST("try_" #f, try_direct<f>)
PyMethodDef g_methods[] = {Q35_FAST("bind", bind),       Q35_FAST("direct", direct),   Q35_METHOD(paged_kv_append),
                           Q35_METHOD(paged_kv_rows),    Q35_METHOD(gated_attn_paged), Q35_METHOD(verify_drafts),
                           Q35_FAST("bind_sampling", bind_sampling), Q35_METHOD(gated_attn_paged_shared),
                           Q35_METHOD(sample_tokens), Q35_METHOD(filter_logits), Q35_METHOD(quantize_rows_i8),
                           Q35_METHOD(add_rmsnorm_i8_), Q35_METHOD(gemm_i8_),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_host() { return PyModule_Create(&g_module); }
