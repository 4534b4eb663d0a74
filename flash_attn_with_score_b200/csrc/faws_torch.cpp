// The operators' plain calls from Python: checks, output tensors, the problem struct and the C entry point in one native
// call; of attention_with_window the autograd function as well.  A call is plain when every tensor is an ordinary strided CUDA tensor that TMA can address, on the current device,
// outside of torch's function and dispatch modes, and the shapes fit; for any other the function returns None and the caller goes
// through the Python path, which words the errors.  What a call computes is the same either way.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "faws.h"

namespace {

constexpr int kOpScoresOnly = 100;  // compute_attention_scores, which has no workspace and no operator id

bool usual_cuda(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const c10::DispatchKeySet keys = THPVariable_Unpack(o).key_set();
  static const c10::DispatchKeySet usual =
      c10::DispatchKeySet(c10::DispatchKey::CUDA) | c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) |
      c10::DispatchKeySet(c10::DispatchKey::AutocastCUDA) | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView);
  return (keys.raw_repr() & ~usual.raw_repr()) == 0 && keys.has(c10::DispatchKey::CUDA);
}

bool plain(PyObject* o) {
  if (!usual_cuda(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 4 || (t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16)) return false;
  if (t.numel() == 0 || t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0) return false;
  return t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && t.stride(2) % 8 == 0;
}

faws_tensor view(const at::Tensor& t) {
  return faws_tensor{const_cast<void*>(t.const_data_ptr()), t.stride(0), t.stride(1), t.stride(2)};
}

bool modes_on() { return at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set(); }

// Shapes, types and devices of q, k, v as every operator wants them, and the problem they make; false where the long way is to see them.
bool plain_problem(PyObject* const* a, faws_problem* p) {
  if (!plain(a[0]) || !plain(a[1]) || !plain(a[2]) || modes_on()) return false;
  const at::Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
  const int64_t B = q.size(0), H = q.size(1), M = q.size(2), D = q.size(3), Hk = k.size(1), N = k.size(2);
  if (k.size(3) != D || v.size(3) != D || (D != 16 && D != 32 && D != 64 && D != 128)) return false;
  if (v.size(1) != Hk || H % Hk != 0 || k.size(0) != B || v.size(0) != B || v.size(2) != N) return false;
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) return false;
  if (B > INT32_MAX || H > INT32_MAX || M > INT32_MAX || N > INT32_MAX) return false;
  const c10::Device dev = q.device();
  if (k.device() != dev || v.device() != dev || dev.index() != c10::cuda::current_device()) return false;
  p->B = (int32_t)B; p->Hq = (int32_t)H; p->Hk = (int32_t)Hk; p->M = (int32_t)M; p->N = (int32_t)N; p->D = (int32_t)D;
  p->dtype = q.scalar_type() == at::kHalf ? FAWS_FP16 : FAWS_BF16;
  p->sm_scale = (float)(1.0 / std::sqrt((double)D));
  p->m_end = (int32_t)M;
  p->q = view(q); p->k = view(k); p->v = view(v);
  return true;
}

// What Python's float() takes of sm_scale (None: as it is); false where that is for the long way to say.
bool scale_of(PyObject* o, float* scale) {
  if (o == Py_None) return true;
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  *scale = (float)x;
  return true;
}

void* current_stream(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

at::Tensor bytes_like(const at::Tensor& t, size_t n) {
  return at::empty({(int64_t)n}, t.options().dtype(at::kByte).requires_grad(false));
}

void check(int st, const char* name) {
  TORCH_CHECK(st == FAWS_OK, name, ": libfaws status ", st, ": ", faws_strerror(st));
}

// attention_with_window's forward pass: out, and the log-normaliser where asked for.
std::pair<at::Tensor, at::Tensor> window_forward(faws_problem& p, const at::Tensor& q, int32_t window, int32_t sinks, bool need_L) {
  at::Tensor out = at::empty_like(q), L, ws;
  p.causal = 1;
  p.out = view(out);
  if (need_L) {
    L = at::empty({p.B, p.Hq, p.M}, q.options().dtype(at::kFloat).requires_grad(false));
    p.log_normalizer = L.data_ptr<float>();
  }
  const int32_t n_splits = faws_window_split_plan(&p, window, sinks);
  const size_t n = n_splits > 1 ? faws_workspace_bytes(FAWS_OP_ATTENTION_SPLIT_KV, &p, n_splits) : 0;
  if (n > 0) ws = bytes_like(q, n);
  check(faws_attention_with_window(&p, window, sinks, n_splits, n > 0 ? ws.data_ptr() : nullptr, n, current_stream(q)),
        "faws_attention_with_window");
  return {out, L};
}

// The same under autograd (the counterpart of api._WindowFunction).
struct WindowFunction : public torch::autograd::Function<WindowFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& v, faws_problem p, int64_t window, int64_t sinks) {
    auto [out, L] = window_forward(p, q, (int32_t)window, (int32_t)sinks, true);
    ctx->save_for_backward({q, k, v, out, L});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = (double)p.sm_scale;
    ctx->mark_non_differentiable({L});
    ctx->set_materialize_grads(false);
    return {out, L};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "attention_with_window has no second derivative (create_graph)");
    auto saved = ctx->get_saved_variables();
    // (a saved-tensor hook may have brought back other tensors than were saved: strides are those of now)
    for (int i = 0; i < 4; ++i)
      if (saved[i].dim() == 4 && saved[i].stride(3) != 1) saved[i] = saved[i].contiguous();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &L = saved[4];
    const at::Tensor none;
    if (grads[0].defined()) {
      const at::Tensor& g = grads[0];
      auto like = [&](const at::Tensor& t) { return t.dim() == 4 && t.scalar_type() == g.scalar_type() && t.device() == g.device(); };
      const bool same = like(q) && like(k) && like(v) && like(out) && q.sizes() == g.sizes() && out.sizes() == g.sizes() &&
                        v.sizes() == k.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3) && k.size(1) > 0 &&
                        q.size(1) % k.size(1) == 0 && L.sizes() == q.sizes().slice(0, 3) && L.scalar_type() == at::kFloat &&
                        L.device() == g.device();
      TORCH_CHECK(same, "attention_with_window: a saved tensor came back with another shape, type or device");
    }
    if (!grads[0].defined()) return {at::zeros_like(q), at::zeros_like(k), at::zeros_like(v), none, none, none};
    const at::Tensor dout = grads[0].stride(3) == 1 ? grads[0] : grads[0].contiguous();
    at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    faws_problem p{};
    p.B = (int32_t)q.size(0); p.Hq = (int32_t)q.size(1); p.Hk = (int32_t)k.size(1);
    p.M = p.m_end = (int32_t)q.size(2); p.N = (int32_t)k.size(2); p.D = (int32_t)q.size(3);
    p.dtype = q.scalar_type() == at::kHalf ? FAWS_FP16 : FAWS_BF16;
    p.causal = 1;
    p.sm_scale = (float)ctx->saved_data["scale"].toDouble();
    p.q = view(q); p.k = view(k); p.v = view(v); p.out = view(out);
    const at::Tensor Lc = L.contiguous();
    p.log_normalizer = Lc.data_ptr<float>();
    const faws_grads g{view(dout), view(dq), view(dk), view(dv)};
    const int32_t window = (int32_t)ctx->saved_data["window"].toInt(), sinks = (int32_t)ctx->saved_data["sinks"].toInt();
    const size_t n = faws_window_backward_bytes(&p, window, sinks);
    const at::Tensor ws = bytes_like(q, n);
    check(faws_attention_with_window_backward(&p, &g, window, sinks, ws.data_ptr(), n, current_stream(q)),
          "faws_attention_with_window_backward");
    return {dq, dk, dv, none, none, none};
  }
};

PyObject* wrap(at::Tensor first, at::Tensor second) {
  if (!second.defined()) return THPVariable_Wrap(std::move(first));
  PyObject* a = THPVariable_Wrap(std::move(first));
  if (a == nullptr) return nullptr;
  PyObject* b = THPVariable_Wrap(std::move(second));
  PyObject* both = b == nullptr ? nullptr : PyTuple_New(2);
  if (both == nullptr) {
    Py_DECREF(a);
    Py_XDECREF(b);
    return nullptr;
  }
  PyTuple_SET_ITEM(both, 0, a);
  PyTuple_SET_ITEM(both, 1, b);
  return both;
}

// window(q, k, v, window, sinks, sm_scale, want_L) -> out, (out, L) or None
PyObject* window(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "window takes seven arguments");
    return nullptr;
  }
  faws_problem p{};
  if (!plain_problem(a, &p) || !scale_of(a[5], &p.sm_scale)) Py_RETURN_NONE;
  const long w = PyLong_AsLong(a[3]), sinks = PyLong_AsLong(a[4]);  // (the caller has bounded both)
  if (PyErr_Occurred()) return nullptr;
  const int want_L = PyObject_IsTrue(a[6]);
  if (want_L < 0) return nullptr;
  const at::Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]), &v = THPVariable_Unpack(a[2]);
  at::Tensor out, L;
  {
    pybind11::gil_scoped_release no_gil;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      const auto both = WindowFunction::apply(q, k, v, p, (int64_t)w, (int64_t)sinks);
      out = both[0];
      L = both[1];
    } else {
      std::tie(out, L) = window_forward(p, q, (int32_t)w, (int32_t)sinks, want_L != 0);
    }
  }
  return wrap(std::move(out), want_L ? std::move(L) : at::Tensor());
  END_HANDLE_TH_ERRORS
}

// Runs a call that launches, without Python's lock: it waits where the launch queue is full.
template <typename Call>
int unlocked(Call call) {
  pybind11::gil_scoped_release no_gil;
  return call();
}

// The page table and lengths of a cache's call as the kernels take them, for B sequences on `dev`.
bool plain_batch(PyObject* table, PyObject* lengths, int64_t B, c10::Device dev, faws_cache_batch* out) {
  if (!usual_cuda(table) || !usual_cuda(lengths)) return false;
  const at::Tensor &t = THPVariable_Unpack(table), &l = THPVariable_Unpack(lengths);
  if (t.dim() != 2 || l.dim() != 1 || t.scalar_type() != at::kInt || l.scalar_type() != at::kInt) return false;
  if (t.size(0) != B || l.size(0) != B || t.size(1) < 1 || t.size(1) > INT32_MAX || B > INT32_MAX) return false;
  if (t.stride(1) != 1 || t.stride(0) < 0 || !l.is_contiguous() || t.device() != dev || l.device() != dev) return false;
  *out = faws_cache_batch{static_cast<const int32_t*>(t.const_data_ptr()), static_cast<const int32_t*>(l.const_data_ptr()),
                          t.stride(0), (int32_t)B, (int32_t)t.size(1)};
  return true;
}

// The cache (the address of its faws_kv_cache) on the device with index `index`; null with an error set.
const faws_kv_cache* cache_of(PyObject* address, PyObject* index, c10::Device* dev) {
  const auto* c = static_cast<const faws_kv_cache*>(PyLong_AsVoidPtr(address));
  const long at = PyLong_AsLong(index);
  if (PyErr_Occurred()) return nullptr;
  *dev = c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)at);
  if (c == nullptr) PyErr_SetString(PyExc_ValueError, "no cache");
  return c;
}
at::ScalarType cache_type(const faws_kv_cache* c) { return c->dtype == FAWS_FP16 ? at::kHalf : at::kBFloat16; }

// cache_write(cache, device, k, v, page_table, lengths) -> True or None
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "cache_write takes six arguments");
    return nullptr;
  }
  c10::Device dev(c10::DeviceType::CUDA, 0);
  const faws_kv_cache* c = cache_of(a[0], a[1], &dev);
  if (c == nullptr) return nullptr;
  if (!plain(a[2]) || !plain(a[3]) || modes_on() || dev.index() != c10::cuda::current_device()) Py_RETURN_NONE;
  const at::Tensor &k = THPVariable_Unpack(a[2]), &v = THPVariable_Unpack(a[3]);
  if ((k.requires_grad() || v.requires_grad()) && at::GradMode::is_enabled()) Py_RETURN_NONE;
  if (k.sizes() != v.sizes() || k.size(1) != c->Hk || k.size(3) != c->D || k.size(2) > INT32_MAX) Py_RETURN_NONE;
  if (k.scalar_type() != cache_type(c) || v.scalar_type() != cache_type(c) || k.device() != dev || v.device() != dev) Py_RETURN_NONE;
  faws_cache_batch b;
  if (!plain_batch(a[4], a[5], k.size(0), dev, &b)) Py_RETURN_NONE;
  const faws_tensor kt = view(k), vt = view(v);
  void* stream = current_stream(k);
  const int32_t rows = (int32_t)k.size(2);
  check(unlocked([&] { return faws_kv_cache_write(c, &b, &kt, &vt, rows, stream); }), "faws_kv_cache_write");
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// cache_read(cache, device, page_table, lengths, rows) -> (k, v) or None
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "cache_read takes five arguments");
    return nullptr;
  }
  c10::Device dev(c10::DeviceType::CUDA, 0);
  const faws_kv_cache* c = cache_of(a[0], a[1], &dev);
  if (c == nullptr) return nullptr;
  const long rows = PyLong_Check(a[4]) ? PyLong_AsLong(a[4]) : 0;
  if (PyErr_Occurred()) return nullptr;
  if (rows < 1 || rows > INT32_MAX || !usual_cuda(a[3]) || modes_on() || dev.index() != c10::cuda::current_device()) Py_RETURN_NONE;
  const at::Tensor& l = THPVariable_Unpack(a[3]);
  faws_cache_batch b;
  if (l.dim() != 1 || l.size(0) < 1 || !plain_batch(a[2], a[3], l.size(0), dev, &b)) Py_RETURN_NONE;
  const auto options = l.options().dtype(cache_type(c)).requires_grad(false);
  at::Tensor k = at::empty({l.size(0), c->Hk, rows, c->D}, options), v = at::empty({l.size(0), c->Hk, rows, c->D}, options);
  const faws_tensor kt = view(k), vt = view(v);
  void* stream = current_stream(k);
  check(unlocked([&] { return faws_kv_cache_read(c, &b, &kt, &vt, (int32_t)rows, stream); }), "faws_kv_cache_read");
  return wrap(std::move(k), std::move(v));
  END_HANDLE_TH_ERRORS
}

// cache_attention(cache, device, q, page_table, lengths, window, sinks, sm_scale, want_L) -> out, (out, L) or None; window 0: none
PyObject* cache_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "cache_attention takes nine arguments");
    return nullptr;
  }
  c10::Device dev(c10::DeviceType::CUDA, 0);
  const faws_kv_cache* c = cache_of(a[0], a[1], &dev);
  if (c == nullptr) return nullptr;
  const long window = PyLong_AsLong(a[5]), sinks = PyLong_AsLong(a[6]);  // (the caller has bounded both)
  const int want_L = PyObject_IsTrue(a[8]);
  if (PyErr_Occurred()) return nullptr;
  if (!plain(a[2]) || modes_on() || dev.index() != c10::cuda::current_device()) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a[2]);
  if (q.requires_grad() && at::GradMode::is_enabled()) Py_RETURN_NONE;
  if (q.size(3) != c->D || q.size(1) % c->Hk != 0 || q.scalar_type() != cache_type(c) || q.device() != dev) Py_RETURN_NONE;
  faws_cache_batch b;
  faws_problem p{};
  p.sm_scale = (float)(1.0 / std::sqrt((double)c->D));
  if (!plain_batch(a[3], a[4], q.size(0), dev, &b) || !scale_of(a[7], &p.sm_scale)) Py_RETURN_NONE;
  if (q.size(1) > INT32_MAX || q.size(2) > INT32_MAX) Py_RETURN_NONE;
  at::Tensor out = at::empty(q.sizes(), q.options().requires_grad(false)), L;
  p.B = b.B; p.Hq = (int32_t)q.size(1); p.Hk = c->Hk; p.M = p.m_end = (int32_t)q.size(2); p.N = 1; p.D = c->D;
  p.dtype = c->dtype; p.causal = 1;
  p.q = view(q);
  p.out = view(out);
  if (want_L) {
    L = at::empty({p.B, p.Hq, p.M}, q.options().dtype(at::kFloat).requires_grad(false));
    p.log_normalizer = L.data_ptr<float>();
  }
  const size_t bytes = faws_kv_cache_workspace_bytes(&p);
  const at::Tensor ws = bytes_like(q, bytes);
  void *scratch = ws.data_ptr(), *stream = current_stream(q);
  check(unlocked([&] { return faws_attention_with_kv_cache(&p, c, &b, (int32_t)window, (int32_t)sinks, scratch, bytes, stream); }),
        "faws_attention_with_kv_cache");
  return wrap(std::move(out), std::move(L));
  END_HANDLE_TH_ERRORS
}

// call(op, q, k, v, causal, sm_scale, split, per_q_head) -> (out, extra), out, extra or None
PyObject* call(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "call takes eight arguments");
    return nullptr;
  }
  const long op = PyLong_AsLong(a[0]);
  if (op == -1 && PyErr_Occurred()) return nullptr;
  faws_problem p{};
  if (!plain_problem(a + 1, &p)) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a[1]);
  const int64_t B = p.B, H = p.Hq, M = p.M, Hk = p.Hk, N = p.N;
  const int causal = PyObject_IsTrue(a[4]);
  if (causal < 0) return nullptr;
  if (!scale_of(a[5], &p.sm_scale)) Py_RETURN_NONE;
  const long split = PyLong_AsLong(a[6]);
  if (split == -1 && PyErr_Occurred()) return nullptr;
  const int per_q_head = PyObject_IsTrue(a[7]);
  if (per_q_head < 0) return nullptr;

  p.causal = causal;
  at::Tensor out;
  if (op != kOpScoresOnly) {
    out = at::empty_like(q);
    p.out = view(out);
  } else {
    p.out = p.q;
  }
  const auto f32 = q.options().dtype(at::kFloat).requires_grad(false);
  at::Tensor extra, ws;
  size_t ws_bytes = 0;
  auto scratch = [&](int32_t which, int32_t arg) {
    ws_bytes = faws_workspace_bytes(which, &p, arg);
    if (ws_bytes > 0) ws = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte).requires_grad(false));
  };
  auto ws_ptr = [&]() -> void* { return ws_bytes > 0 ? ws.data_ptr() : nullptr; };
  int32_t n_splits = 1;
  const char* name = "";
  switch (op) {
    case FAWS_OP_ATTENTION:
      n_splits = faws_split_kv_plan(&p);
      name = n_splits > 1 ? "faws_attention_split_kv" : "faws_attention";
      if (n_splits > 1) scratch(FAWS_OP_ATTENTION_SPLIT_KV, n_splits);
      break;
    case FAWS_OP_SCORES: name = "faws_attention_with_scores"; extra = at::empty({B, H, M, N}, f32); break;
    case kOpScoresOnly:
      name = "faws_compute_attention_scores";
      extra = at::empty({B, H, M, N}, q.options().requires_grad(false));
      break;
    case FAWS_OP_ROW_SUM: name = "faws_attention_with_row_sum"; extra = at::empty({B, H, M}, f32); break;
    default:
      extra = at::empty({B, per_q_head ? H : Hk, split > 0 ? split : N}, f32);
      scratch((int32_t)op, (int32_t)split);
  }
  void* stream = current_stream(q);
  float* sums = extra.defined() && extra.scalar_type() == at::kFloat ? extra.data_ptr<float>() : nullptr;
  int st = FAWS_EINVAL;
  Py_BEGIN_ALLOW_THREADS
  switch (op) {
    case FAWS_OP_ATTENTION:
      st = n_splits > 1 ? faws_attention_split_kv(&p, n_splits, ws_ptr(), ws_bytes, stream) : faws_attention(&p, stream);
      break;
    case FAWS_OP_SCORES: st = faws_attention_with_scores(&p, sums, FAWS_SCORES_F32, 0xff800000u, stream); break;
    case kOpScoresOnly: st = faws_compute_attention_scores(&p, extra.data_ptr(), FAWS_SCORES_INPUT, stream); break;
    case FAWS_OP_ROW_SUM: st = faws_attention_with_row_sum(&p, sums, stream); break;
    case FAWS_OP_COL_SUM:
      name = "faws_attention_with_col_sum";
      st = faws_attention_with_col_sum(&p, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    case FAWS_OP_COL_SUM_SEQUENTIAL:
      name = "faws_attention_with_col_sum_sequential";
      st = faws_attention_with_col_sum_sequential(&p, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    case FAWS_OP_SOFTMAX_COL_SUM:
      name = "faws_attention_with_softmax_col_sum";
      st = faws_attention_with_softmax_col_sum(&p, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    case FAWS_OP_CROSS_QK_SUM:
      name = "faws_attention_cross_token_qk_sum";
      st = faws_attention_cross_token_qk_sum(&p, (int32_t)split, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    case FAWS_OP_CROSS_SOFTMAX_SUM:
      name = "faws_attention_cross_token_softmax_sum";
      st = faws_attention_cross_token_softmax_sum(&p, (int32_t)split, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    case FAWS_OP_CROSS_SOFTMAX_SUM_BUFFERED:
      name = "faws_attention_cross_token_softmax_sum_buffered";
      st = faws_attention_cross_token_softmax_sum_buffered(&p, (int32_t)split, sums, per_q_head, ws_ptr(), ws_bytes, stream);
      break;
    default: break;
  }
  Py_END_ALLOW_THREADS
  if (st != FAWS_OK) {
    PyErr_Format(PyExc_RuntimeError, "%s: libfaws status %d: %s", name, st, faws_strerror(st));
    return nullptr;
  }
  if (!out.defined()) return THPVariable_Wrap(std::move(extra));
  return wrap(std::move(out), std::move(extra));
  END_HANDLE_TH_ERRORS
}

#define FAWS_FASTCALL(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef kMethods[] = {
    {"window", FAWS_FASTCALL(window), "window(q, k, v, window, sinks, sm_scale, want_L), or None"},
    {"cache_write", FAWS_FASTCALL(cache_write), "cache_write(cache, device, k, v, page_table, lengths): True, or None"},
    {"cache_read", FAWS_FASTCALL(cache_read), "cache_read(cache, device, page_table, lengths, rows), or None"},
    {"cache_attention", FAWS_FASTCALL(cache_attention),
     "cache_attention(cache, device, q, page_table, lengths, window, sinks, sm_scale, want_L), or None"},
    {"call", FAWS_FASTCALL(call),
     "call(op, q, k, v, causal, sm_scale, split, per_q_head): a plain call, or None where it is not one"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_plain", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// Tensors are read by the layout of the torch that this was compiled against, so no other one may load it, and no other
// Python.
PyMODINIT_FUNC PyInit__plain() {
#define FAWS_STR2(x) #x
#define FAWS_STR(x) FAWS_STR2(x)
  static const char python[] = FAWS_STR(PY_MAJOR_VERSION) "." FAWS_STR(PY_MINOR_VERSION) ".";
  if (std::strncmp(Py_GetVersion(), python, sizeof(python) - 1) != 0) {
    PyErr_Format(PyExc_ImportError, "_plain.so was built for Python %s, this is %s", python, Py_GetVersion());
    return nullptr;
  }
  PyObject* torch = PyImport_ImportModule("torch");
  if (torch == nullptr) return nullptr;
  PyObject* version = PyObject_GetAttrString(torch, "__version__");
  Py_DECREF(torch);
  if (version == nullptr) return nullptr;
  const bool same = PyUnicode_Check(version) && PyUnicode_CompareWithASCIIString(version, FAWS_TORCH_VERSION) == 0;
  if (!same) PyErr_Format(PyExc_ImportError, "_plain.so was built for torch " FAWS_TORCH_VERSION ", this is %S", version);
  Py_DECREF(version);
  return same ? PyModule_Create(&kModule) : nullptr;
}
