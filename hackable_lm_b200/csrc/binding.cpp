// Python binding of the 8-bit operators (module hackable_lm_b200._hlm_torch): argument
// checks, output allocation and the C ABI call of one operator in one C call.
//
// The kernels of a few tokens run for 2 us; the same steps in Python with ctypes cost
// 10 to 18 us a call, here 0.6 to 2 beside the launch itself (2.5).
//
// Every function returns None, and does nothing, when its tensors are not plain ones that
// may go straight to the library: not on CUDA, a tensor subclass, wrapped by a transform,
// under a dispatch mode or torch.jit.trace, or with a gradient asked for.  The caller then goes through the
// registered operator.  The entry points of libhlm_b200 are handed over by address
// (set_entry_points), so that the one library that ctypes loaded is used.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <string>

#include "../../include/hlm_b200.h"

namespace {

decltype(&hlm_strerror) p_strerror = nullptr;
decltype(&hlm_quantize_rows) p_quantize_rows = nullptr;
decltype(&hlm_dequantize_rows) p_dequantize_rows = nullptr;
decltype(&hlm_residual_rms_norm_q8) p_residual_rms_norm_q8 = nullptr;
decltype(&hlm_linear_q8) p_linear_q8 = nullptr;
decltype(&hlm_swiglu_ckpt8_fwd) p_swiglu_ckpt8_fwd = nullptr;
decltype(&hlm_swiglu_ckpt8_bwd) p_swiglu_ckpt8_bwd = nullptr;
decltype(&hlm_weight_grad_q8) p_weight_grad_q8 = nullptr;
decltype(&hlm_weight_grad_q8_workspace_bytes) p_weight_grad_q8_workspace_bytes = nullptr;
PyObject* g_error = nullptr;  // _lib.HlmError

constexpr int64_t kGroup = 128;

const c10::DispatchKeySet kWrapped({
    c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::BatchedNestedTensor,
    c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched, c10::DispatchKey::Functionalize,
    c10::DispatchKey::Conjugate, c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});

// The tensor behind a Python object that may go straight to the library, or null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.key_set().has_any(kWrapped)) return nullptr;
  if (t.requires_grad() && c10::GradMode::is_enabled()) return nullptr;
  // no operator here has a forward-mode derivative, and the registered ones would drop the tangent
  TORCH_CHECK(!t._fw_grad(0).defined(), "hackable_lm_b200: the 8-bit operators have no forward-mode derivatives");
  return &t;
}

bool modes_active() {
  return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::tracer::impl::is_dispatch_enabled();
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return HLM_F32;
    case at::kBFloat16:
      return HLM_BF16;
    case at::kHalf:
      return HLM_F16;
    default:
      TORCH_CHECK(false, "hackable_lm_b200: unsupported dtype ", t);
  }
}
at::ScalarType dtype_of(int code) {
  return code == HLM_F32 ? at::kFloat : code == HLM_BF16 ? at::kBFloat16 : at::kHalf;
}

void same_device(const at::Tensor& a, std::initializer_list<const at::Tensor*> others) {
  for (const at::Tensor* t : others)
    TORCH_CHECK(t == nullptr || t->device() == a.device(),
                "hackable_lm_b200: all tensors must be on the same device");
}

// Contiguous and 16-byte aligned, as the tensor-core kernels read it (a copy where it is not).
at::Tensor packed(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}

// An uninitialised tensor on t's device (at::empty less its way through the dispatcher, 0.3 us of each).
at::Tensor fresh(const at::Tensor& t, c10::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}

std::vector<int64_t> with_last(const at::Tensor& t, int64_t last) {
  std::vector<int64_t> v = t.sizes().vec();
  v.back() = last;
  return v;
}

void check_rows(const char* what, const at::Tensor& q, const at::Tensor& scale) {
  TORCH_CHECK(q.scalar_type() == at::kChar && scale.scalar_type() == at::kFloat && q.dim() >= 1 &&
                  scale.sizes() == q.sizes().slice(0, q.dim() - 1),
              what, ": needs int8 codes [..., C] and their fp32 scales [...], got ", q.scalar_type(), " ", q.sizes(),
              " and ", scale.scalar_type(), " ", scale.sizes());
}
void check_cols(const char* what, const at::Tensor& x) {
  dtype_code(x.scalar_type());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": needs at least one column, got shape ", x.sizes());
}

struct LibraryError {
  std::string text;
};
void check_rc(int rc, const char* name) {
  if (rc != HLM_OK)
    throw LibraryError{std::string(name) + " failed: " + p_strerror(rc) + " (code " + std::to_string(rc) + ")"};
}

// The current stream of t's device, which is made current for the scope, with the
// interpreter lock released: a launch waits while the stream's queue is full, and what it
// waits for may be another Python thread's.  done() takes the lock again before a result
// is made; an exception takes it on its way out.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  PyThreadState* thread;
  explicit On(const at::Tensor& t) {
    if (c10::cuda::current_device() != t.get_device()) guard.set_device(t.device());
    stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
    thread = PyEval_SaveThread();
  }
  On(const On&) = delete;
  void done() {
    if (thread != nullptr) PyEval_RestoreThread(thread);
    thread = nullptr;
  }
  ~On() { done(); }
};

template <class F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const LibraryError& e) {
    PyErr_SetString(g_error != nullptr ? g_error : PyExc_RuntimeError, e.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* pack(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = THPVariable_Wrap(t);
    if (o == nullptr) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

bool arity(const char* name, Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
  return false;
}

#define RETURN_NONE_UNLESS(cond) \
  do {                           \
    if (!(cond)) Py_RETURN_NONE; \
  } while (0)

PyObject* quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("quantize_rows", n, 1)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* x0 = plain(a[0]);
    RETURN_NONE_UNLESS(x0 != nullptr && !modes_active());
    check_cols("quantize_rows", *x0);
    On on(*x0);
    const at::Tensor x = x0->contiguous();
    at::Tensor q = fresh(x, x.sizes(), at::kChar);
    at::Tensor scale = fresh(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    check_rc(p_quantize_rows(x.const_data_ptr(), q.data_ptr(), scale.data_ptr<float>(), scale.numel(), x.size(-1),
                             dtype_code(x.scalar_type()), on.stream),
             "hlm_quantize_rows");
    on.done();
    return pack({q, scale});
  });
}

PyObject* dequantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("dequantize_rows", n, 3)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q0 = plain(a[0]), *s0 = plain(a[1]);
    RETURN_NONE_UNLESS(q0 != nullptr && s0 != nullptr && !modes_active());
    const int code = static_cast<int>(PyLong_AsLong(a[2]));
    check_rows("dequantize_rows", *q0, *s0);
    same_device(*q0, {s0});
    On on(*q0);
    const at::Tensor q = q0->contiguous(), scale = s0->contiguous();
    at::Tensor out = fresh(q, q.sizes(), dtype_of(code));
    if (q.numel() > 0)
      check_rc(p_dequantize_rows(q.const_data_ptr(), scale.const_data_ptr<float>(), out.data_ptr(), scale.numel(),
                                 q.size(-1), code, on.stream),
               "hlm_dequantize_rows");
    on.done();
    return THPVariable_Wrap(out);
  });
}

// residual (or None), branch, weight (or None), eps -> (out, q, scale) or (q, scale)
PyObject* residual_rms_norm_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("residual_rms_norm_q8", n, 4)) return nullptr;
  return guarded([&]() -> PyObject* {
    const bool has_r = a[0] != Py_None, has_w = a[2] != Py_None;
    const char* what = has_r ? "residual_rms_norm_q8" : "rms_norm_q8";
    const at::Tensor* x0 = plain(a[1]);
    const at::Tensor* r0 = has_r ? plain(a[0]) : nullptr;
    const at::Tensor* w0 = has_w ? plain(a[2]) : nullptr;
    RETURN_NONE_UNLESS(x0 != nullptr && (!has_r || r0 != nullptr) && (!has_w || w0 != nullptr) && !modes_active());
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    check_cols(what, *x0);
    same_device(*x0, {r0, w0});
    TORCH_CHECK(!has_r || (r0->sizes() == x0->sizes() && r0->scalar_type() == x0->scalar_type()), what,
                ": residual and branch must match in shape and dtype");
    TORCH_CHECK(!has_w || (w0->dim() == 1 && w0->size(0) == x0->size(-1)), what, ": weight must be [", x0->size(-1), "]");
    On on(*x0);
    const at::Tensor x = x0->contiguous();
    const at::Tensor r = has_r ? r0->contiguous() : at::Tensor();
    const at::Tensor w = has_w ? w0->to(x.scalar_type()).contiguous() : at::Tensor();
    at::Tensor out = has_r ? fresh(x, x.sizes(), x.scalar_type()) : at::Tensor();
    at::Tensor q = fresh(x, x.sizes(), at::kChar);
    at::Tensor scale = fresh(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    check_rc(p_residual_rms_norm_q8(has_r ? r.const_data_ptr() : nullptr, x.const_data_ptr(),
                                    has_w ? w.const_data_ptr() : nullptr, has_r ? out.data_ptr() : nullptr,
                                    q.data_ptr(), scale.data_ptr<float>(), scale.numel(), x.size(-1),
                                    static_cast<float>(eps), dtype_code(x.scalar_type()), on.stream),
             "hlm_residual_rms_norm_q8");
    on.done();
    return has_r ? pack({out, q, scale}) : pack({q, scale});
  });
}

PyObject* linear_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("linear_q8", n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q0 = plain(a[0]), *s0 = plain(a[1]), *w0 = plain(a[2]), *t0 = plain(a[3]);
    RETURN_NONE_UNLESS(q0 != nullptr && s0 != nullptr && w0 != nullptr && t0 != nullptr && !modes_active());
    const int code = static_cast<int>(PyLong_AsLong(a[4]));
    check_rows("linear_q8", *q0, *s0);
    check_rows("linear_q8 (weight)", *w0, *t0);
    TORCH_CHECK(w0->dim() == 2 && w0->size(1) == q0->size(-1), "linear_q8: weight must be [N, ", q0->size(-1), "], got ",
                w0->sizes());
    same_device(*q0, {s0, w0, t0});
    On on(*q0);
    const at::Tensor q = packed(*q0), w = packed(*w0), scale = s0->contiguous(), w_scale = t0->contiguous();
    const int64_t N = w.size(0), K = w.size(1);
    at::Tensor out = fresh(q, with_last(q, N), dtype_of(code));
    check_rc(p_linear_q8(q.const_data_ptr(), scale.const_data_ptr<float>(), w.const_data_ptr(),
                         w_scale.const_data_ptr<float>(), out.data_ptr(), scale.numel(), N, K, code, on.stream),
             "hlm_linear_q8");
    on.done();
    return THPVariable_Wrap(out);
  });
}

int64_t check_gate_up(const char* what, const at::Tensor& t) {
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) % 2 == 0, what, ": the last dimension must be even (gate | up), got shape ",
              t.sizes());
  return t.size(-1) / 2;
}
int64_t scale_cols(int64_t hidden) { return 2 * ((hidden + kGroup - 1) / kGroup); }

PyObject* swiglu_ckpt8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("swiglu_ckpt8", n, 1)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* x0 = plain(a[0]);
    RETURN_NONE_UNLESS(x0 != nullptr && !modes_active());
    const int code = dtype_code(x0->scalar_type());
    const int64_t hidden = check_gate_up("swiglu_ckpt8", *x0);
    On on(*x0);
    const at::Tensor x = x0->contiguous();
    at::Tensor h = fresh(x, with_last(x, hidden), x.scalar_type());
    at::Tensor q = fresh(x, x.sizes(), at::kChar);
    at::Tensor scale = fresh(x, with_last(x, scale_cols(hidden)), at::kFloat);
    if (hidden > 0)
      check_rc(p_swiglu_ckpt8_fwd(x.const_data_ptr(), h.data_ptr(), q.data_ptr(), scale.data_ptr<float>(),
                                  h.numel() / hidden, hidden, code, on.stream),
               "hlm_swiglu_ckpt8_fwd");
    on.done();
    return pack({h, q, scale});
  });
}

PyObject* swiglu_ckpt8_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("swiglu_ckpt8_backward", n, 3)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *q0 = plain(a[0]), *s0 = plain(a[1]), *g0 = plain(a[2]);
    RETURN_NONE_UNLESS(q0 != nullptr && s0 != nullptr && g0 != nullptr && !modes_active());
    const int code = dtype_code(g0->scalar_type());
    const int64_t hidden = check_gate_up("swiglu_ckpt8_backward", *q0);
    TORCH_CHECK(q0->scalar_type() == at::kChar && s0->scalar_type() == at::kFloat &&
                    g0->sizes() == c10::IntArrayRef(with_last(*q0, hidden)) &&
                    s0->sizes() == c10::IntArrayRef(with_last(*q0, scale_cols(hidden))),
                "swiglu_ckpt8_backward: needs the codes and scales of swiglu_ckpt8 and a gradient [..., ", hidden,
                "], got ", q0->sizes(), ", ", s0->sizes(), ", ", g0->sizes());
    same_device(*q0, {s0, g0});
    On on(*q0);
    const at::Tensor q = q0->contiguous(), scale = s0->contiguous(), g = g0->contiguous();
    at::Tensor grad = fresh(g, q.sizes(), g.scalar_type());
    if (hidden > 0)
      check_rc(p_swiglu_ckpt8_bwd(q.const_data_ptr(), scale.const_data_ptr<float>(), g.const_data_ptr(),
                                  grad.data_ptr(), g.numel() / hidden, hidden, code, on.stream),
               "hlm_swiglu_ckpt8_bwd");
    on.done();
    return THPVariable_Wrap(grad);
  });
}

PyObject* weight_grad_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("weight_grad_q8", n, 3)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *g0 = plain(a[0]), *q0 = plain(a[1]), *s0 = plain(a[2]);
    RETURN_NONE_UNLESS(g0 != nullptr && q0 != nullptr && s0 != nullptr && !modes_active());
    check_rows("weight_grad_q8", *q0, *s0);
    TORCH_CHECK(g0->scalar_type() == at::kBFloat16 || g0->scalar_type() == at::kHalf,
                "weight_grad_q8: grad must be bf16 or fp16, got ", g0->scalar_type());
    TORCH_CHECK(g0->dim() >= 1 && g0->sizes().slice(0, g0->dim() - 1) == q0->sizes().slice(0, q0->dim() - 1),
                "weight_grad_q8: grad [..., N] and the codes [..., K] must have the same rows, got ", g0->sizes(), " and ",
                q0->sizes());
    same_device(*g0, {q0, s0});
    On on(*g0);
    const at::Tensor g = packed(*g0), q = packed(*q0), scale = s0->contiguous();
    const int64_t tokens = scale.numel(), N = g.size(-1), K = q.size(-1);
    at::Tensor out = fresh(g, {N, K}, g.scalar_type());
    const size_t bytes = p_weight_grad_q8_workspace_bytes(tokens, N, K);
    at::Tensor ws = fresh(g, {static_cast<int64_t>(bytes)}, at::kByte);
    check_rc(p_weight_grad_q8(g.const_data_ptr(), q.const_data_ptr(), scale.const_data_ptr<float>(), out.data_ptr(),
                              ws.data_ptr(), bytes, tokens, N, K, dtype_code(g.scalar_type()), on.stream),
             "hlm_weight_grad_q8");
    on.done();
    return THPVariable_Wrap(out);
  });
}

// {name: address} of libhlm_b200's entry points, and the exception for its error codes.
PyObject* set_entry_points(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arity("set_entry_points", n, 2)) return nullptr;
  auto take = [&](const char* name, auto& p) {
    PyObject* o = PyDict_GetItemString(a[0], name);
    if (o == nullptr) {
      PyErr_Format(PyExc_KeyError, "%s", name);
      return false;
    }
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(PyLong_AsVoidPtr(o));
    return p != nullptr;
  };
  if (!take("hlm_strerror", p_strerror) || !take("hlm_quantize_rows", p_quantize_rows) ||
      !take("hlm_dequantize_rows", p_dequantize_rows) || !take("hlm_residual_rms_norm_q8", p_residual_rms_norm_q8) ||
      !take("hlm_linear_q8", p_linear_q8) || !take("hlm_swiglu_ckpt8_fwd", p_swiglu_ckpt8_fwd) ||
      !take("hlm_swiglu_ckpt8_bwd", p_swiglu_ckpt8_bwd) || !take("hlm_weight_grad_q8", p_weight_grad_q8) ||
      !take("hlm_weight_grad_q8_workspace_bytes", p_weight_grad_q8_workspace_bytes))
    return nullptr;
  Py_INCREF(a[1]);
  Py_XDECREF(g_error);
  g_error = a[1];
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {METHOD(quantize_rows), METHOD(dequantize_rows), METHOD(residual_rms_norm_q8),
                          METHOD(linear_q8), METHOD(swiglu_ckpt8), METHOD(swiglu_ckpt8_backward),
                          METHOD(weight_grad_q8), METHOD(set_entry_points), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_hlm_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hlm_torch(void) { return PyModule_Create(&kModule); }
