// CPython binding of the operators in ops.py for the calls that a training or serving loop repeats:
// argument checks, allocation of the result, the C entry point and the autograd node in one native
// call.  A small product takes 3 to 5 microseconds on the GPU; the same steps in Python take 10 on
// the host.  The entry points are passed in as addresses (bind), so this module works with whichever
// build of the library ops.py has loaded.
//
// A function returns its result, or None where its arguments do not fit: ops.py then says what is wrong.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>

#include <unordered_set>
#include <vector>

#include "../../include/fused_moe_c.h"

namespace {

struct {
  decltype(&fmoe_grouped_matmul) grouped = nullptr;
  decltype(&fmoe_grouped_matmul_wgrad) wgrad = nullptr;
  decltype(&fmoe_matmul_block128) block128 = nullptr;
  decltype(&fmoe_silu_mul) silu = nullptr;
  decltype(&fmoe_silu_mul_quantise) silu_quantise = nullptr;
  decltype(&fmoe_silu_mul_backward) silu_backward = nullptr;
  decltype(&fmoe_last_error) last_error = nullptr;
} F;
PyObject* g_error_class = nullptr;      // FmoeError(code, text)

// What an entry point reported.
struct Failure : std::runtime_error {
  int code;
  Failure(int rc, const char* text) : std::runtime_error(text), code(rc) {}
};

bool aligned(const at::Tensor& t, uintptr_t to) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (to - 1)) == 0; }
// A dense tensor on a CUDA device.
bool dense(const at::Tensor& t, uintptr_t to = 16) {
  return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && aligned(t, to);
}
bool half_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
int dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? FMOE_BF16 : FMOE_F16; }
bool byte_type(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kByte; }
void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
void check(int rc) {
  if (rc != FMOE_OK) throw Failure(rc, F.last_error());
}

// The interpreter's lock is not held while a call allocates and launches: either may wait for the GPU.
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

bool fits32(const at::Tensor& t) {
  for (const int64_t d : t.sizes())
    if (d > INT32_MAX) return false;
  return true;
}
// Forward-mode derivatives go by a mode of their own: torch.no_grad does not switch them off.
void refuse_tangent(const at::Tensor& t) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    throw Failure(FMOE_ERR_INVALID_ARG, "forward-mode derivatives are not supported");
}

// True while a tracer records what runs (make_fx, torch.jit.trace, export): it would see the allocation of
// the result and nothing else.  Inside a registered operator, whose call it records, it is off.
bool traced() {
  auto on = [](at::DispatchKey k) { return c10::impl::tls_is_dispatch_key_included(k) && !c10::impl::tls_is_dispatch_key_excluded(k); };
  return c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() ||
         on(at::DispatchKey::Tracer) || on(at::DispatchKey::PreDispatch);
}

// A backward pass is traced as a call is: the recorded program would hold empty gradients.
void refuse_traced_backward() {
  if (traced())
    throw Failure(FMOE_ERR_INVALID_ARG, "a traced program cannot hold this backward pass: use torch.ops.therock_b200 (import therock_b200.torch_op)");
}

// A backward pass that is being captured cannot hand gradients to a node of the default stream, which
// cannot join a capture: a leaf has such a node as long as any earlier graph of it lives.  The engine
// would break the capture, and with it the process; this ends the pass with an error instead.  It looks
// at every node that the rest of this pass reaches from here, and at no other.
void refuse_default_stream_in_capture(int device) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (!node) return;
  const c10::Stream blocked = c10::cuda::getDefaultCUDAStream(static_cast<c10::DeviceIndex>(device)).unwrap();
  std::vector<torch::autograd::Node*> left{node.get()};
  std::unordered_set<torch::autograd::Node*> seen{node.get()};
  while (!left.empty()) {
    torch::autograd::Node* at = left.back();
    left.pop_back();
    for (uint32_t i = 0; i < at->num_outputs(); ++i) {
      if (!at->task_should_compute_output(i)) continue;
      torch::autograd::Node* next = at->next_edge(i).function.get();
      if (!seen.insert(next).second) continue;
      const std::optional<c10::Stream> s = next->stream();
      if (s && *s == blocked)
        throw std::runtime_error(
            "a backward pass is being captured in a CUDA graph while an earlier graph of the same tensors, recorded "
            "on the default stream, is alive: drop its results (or record it on a side stream) before the capture");
      left.push_back(next);
    }
  }
}

// A gradient that autograd may hand over with any strides, or a tensor that a hook on saved tensors gave
// back, as the kernels read it.
at::Tensor for_kernel(const at::Tensor& t, uintptr_t to = 16) {
  at::Tensor c = t.contiguous();
  return aligned(c, to) ? c : c.clone();
}

bool same_kind(const at::Tensor& a, const at::Tensor& b) { return a.scalar_type() == b.scalar_type() && a.get_device() == b.get_device(); }
// What a graph kept comes back through the user's hooks, if there are any, and is checked like an argument.
[[noreturn]] void throw_not_saved() {
  throw Failure(FMOE_ERR_INVALID_ARG, "what came back from a hook on saved tensors is not what was saved (type, shape or device)");
}

// Gradients are first order: what a backward pass with create_graph = True returns raises when it is
// differentiated again.
torch::autograd::variable_list once(torch::autograd::variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list some;
  for (auto& g : grads)
    if (g.defined()) { some.push_back(g.detach()); some.back().requires_grad_(); }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that has first derivatives only", static_cast<int64_t>(some.size()));
  auto out = (*error)(std::move(some));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// ----------------------------------------------------------------------------- products grouped by expert
bool grouped_fits(const at::Tensor& x, const at::Tensor& w, const at::Tensor& off) {
  return dense(x) && dense(w) && dense(off, 4) && fits32(w) && half_type(x.scalar_type()) && w.scalar_type() == x.scalar_type() &&
         off.scalar_type() == at::kInt && x.dim() == 2 && w.dim() == 3 && off.dim() == 1 && w.size(2) == x.size(1) &&
         off.size(0) == w.size(0) + 1 && w.get_device() == x.get_device() && off.get_device() == x.get_device();
}

at::Tensor grouped(const at::Tensor& x, const at::Tensor& w, const at::Tensor& off, bool transpose) {
  at::Tensor out = at::empty({x.size(0), w.size(transpose ? 2 : 1)}, x.options().requires_grad(false));
  check(F.grouped(x.data_ptr(), w.data_ptr(), off.data_ptr<int32_t>(), x.size(0), static_cast<int32_t>(w.size(0)),
                  static_cast<int32_t>(w.size(1)), static_cast<int32_t>(w.size(2)), dtype_code(x), transpose, out.data_ptr(),
                  nullptr, stream_of(x)));
  return out;
}

struct GroupedMatmul : torch::autograd::Function<GroupedMatmul> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& off) {
    ctx->save_for_backward({x, w, off});
    return grouped(x, w, off, false);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    refuse_traced_backward();
    refuse_default_stream_in_capture(grads[0].get_device());
    torch::autograd::variable_list out(3);
    {
      at::NoGradGuard no_grad;
      const at::Tensor dy = for_kernel(grads[0]), x = for_kernel(saved[0]), w = for_kernel(saved[1]), off = for_kernel(saved[2], 4);
      if (!grouped_fits(x, w, off) || !same_kind(x, dy) || dy.size(0) != x.size(0) || dy.size(1) != w.size(1)) throw_not_saved();
      if (ctx->needs_input_grad(0)) out[0] = grouped(dy, w, off, true);
      if (ctx->needs_input_grad(1)) {
        out[1] = at::empty(w.sizes(), w.options().requires_grad(false));
        check(F.wgrad(dy.data_ptr(), x.data_ptr(), off.data_ptr<int32_t>(), x.size(0), static_cast<int32_t>(w.size(0)),
                      static_cast<int32_t>(w.size(1)), static_cast<int32_t>(w.size(2)), dtype_code(x), out[1].data_ptr(),
                      nullptr, stream_of(x)));
      }
    }
    return once(std::move(out));
  }
};

// ----------------------------------------------------------------------------- the gated activation
bool silu_fits(const at::Tensor& gu, const std::optional<at::Tensor>& weight) {
  if (!(dense(gu) && half_type(gu.scalar_type()) && gu.dim() == 2 && gu.size(1) % 16 == 0 && gu.size(1) > 0 &&
        gu.size(1) <= INT32_MAX))
    return false;
  return !weight || (dense(*weight, 4) && weight->scalar_type() == at::kFloat && weight->dim() == 1 &&
                     weight->size(0) == gu.size(0) && weight->get_device() == gu.get_device());
}
const float* weight_ptr(const std::optional<at::Tensor>& w) { return w ? w->data_ptr<float>() : nullptr; }

at::Tensor silu(const at::Tensor& gu, const std::optional<at::Tensor>& weight) {
  const int64_t width = gu.size(1) / 2;
  at::Tensor out = at::empty({gu.size(0), width}, gu.options().requires_grad(false));
  check(F.silu(gu.data_ptr(), weight_ptr(weight), gu.size(0), static_cast<int32_t>(width), dtype_code(gu), out.data_ptr(), stream_of(gu)));
  return out;
}

struct SiluMul : torch::autograd::Function<SiluMul> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& gu, const std::optional<at::Tensor>& weight) {
    ctx->save_for_backward({gu, weight ? *weight : at::Tensor()});
    return silu(gu, weight);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    refuse_traced_backward();
    refuse_default_stream_in_capture(grads[0].get_device());
    torch::autograd::variable_list out(2);
    {
      at::NoGradGuard no_grad;
      const at::Tensor dy = for_kernel(grads[0]), gu = for_kernel(saved[0]);
      const at::Tensor weight = saved[1].defined() ? for_kernel(saved[1], 4) : at::Tensor();
      if (!silu_fits(gu, weight.defined() ? std::optional<at::Tensor>(weight) : std::nullopt) || !same_kind(gu, dy) ||
          dy.size(0) != gu.size(0) || 2 * dy.size(1) != gu.size(1))
        throw_not_saved();
      out[0] = at::empty(gu.sizes(), gu.options().requires_grad(false));
      if (weight.defined()) out[1] = at::empty(weight.sizes(), weight.options().requires_grad(false));
      check(F.silu_backward(gu.data_ptr(), weight.defined() ? weight.data_ptr<float>() : nullptr, dy.data_ptr(), gu.size(0),
                            static_cast<int32_t>(gu.size(1) / 2), dtype_code(gu), out[0].data_ptr(),
                            weight.defined() ? out[1].data_ptr<float>() : nullptr, stream_of(gu)));
    }
    return once(std::move(out));
  }
};

// ----------------------------------------------------------------------------- Python entry points
PyObject* raise(const Failure& f) {
  PyObject* e = PyObject_CallFunction(g_error_class, "is", f.code, f.what());
  if (e != nullptr) {
    PyErr_SetObject(g_error_class, e);
    Py_DECREF(e);
  }
  return nullptr;
}
#define FMOE_TRY HANDLE_TH_ERRORS try {
#define FMOE_CATCH } catch (const Failure& f) { return raise(f); } END_HANDLE_TH_ERRORS

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

PyObject* py_grouped_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FMOE_TRY
  const at::Tensor *x, *w, *off;
  if (n != 3 || traced() || !(x = tensor(args[0])) || !(w = tensor(args[1])) || !(off = tensor(args[2])) || !grouped_fits(*x, *w, *off))
    Py_RETURN_NONE;
  refuse_tangent(*x);
  refuse_tangent(*w);
  at::Tensor out;
  {
    Unlocked unlocked;
    out = at::GradMode::is_enabled() && (x->requires_grad() || w->requires_grad()) ? GroupedMatmul::apply(*x, *w, *off)
                                                                                   : grouped(*x, *w, *off, false);
  }
  return THPVariable_Wrap(std::move(out));
  FMOE_CATCH
}

PyObject* py_matmul_block128(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FMOE_TRY
  const at::Tensor *a, *sa, *w, *sw;
  if (n != 5 || traced() || !(a = tensor(args[0])) || !(sa = tensor(args[1])) || !(w = tensor(args[2])) || !(sw = tensor(args[3]))) Py_RETURN_NONE;
  const bool hw = PyLong_AsLong(args[4]) == FMOE_QUANT_BLOCK128_UE8M0;
  if (!(dense(*a) && dense(*w) && dense(*sa, 4) && dense(*sw, 4) && byte_type(a->scalar_type()) && byte_type(w->scalar_type()) &&
        a->dim() == 2 && w->dim() == 2 && a->size(1) == w->size(1) && sa->dim() == 2 && sw->dim() == 2)) 
    Py_RETURN_NONE;
  const int64_t m = a->size(0), k = a->size(1), nn = w->size(0), kb = k / 128;
  const int64_t row_bytes = hw ? (kb + 3) / 4 * 4 : 4 * kb;
  const bool bytes = sa->scalar_type() == at::kByte, floats = sa->scalar_type() == at::kFloat && !hw;
  if (k % 128 != 0 || k == 0 || nn == 0 || k > INT32_MAX || nn > INT32_MAX || !(bytes || floats) || sa->size(0) != m ||
      sa->size(1) != (bytes ? row_bytes : kb) || sw->scalar_type() != at::kFloat || sw->size(0) != (nn + 127) / 128 || sw->size(1) != kb ||
      sa->get_device() != a->get_device() || w->get_device() != a->get_device() || sw->get_device() != a->get_device())
    Py_RETURN_NONE;
  at::Tensor out;
  {
    Unlocked unlocked;
    out = at::empty({m, nn}, a->options().dtype(at::kBFloat16).requires_grad(false));
    check(F.block128(a->data_ptr(), sa->data_ptr(), w->data_ptr(), sw->data_ptr<float>(), m, static_cast<int32_t>(nn),
                     static_cast<int32_t>(k), hw ? FMOE_QUANT_BLOCK128_UE8M0 : FMOE_QUANT_BLOCK128, out.data_ptr(),
                     nullptr, stream_of(*a)));
  }
  return THPVariable_Wrap(std::move(out));
  FMOE_CATCH
}

// The optional weight of an activation's rows; false where the argument is neither None nor a tensor.
bool weight_of(PyObject* o, std::optional<at::Tensor>* weight) {
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (t) *weight = *t;
  return t != nullptr;
}

PyObject* py_silu_mul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FMOE_TRY
  const at::Tensor* gu;
  std::optional<at::Tensor> weight;
  if (n != 2 || traced() || !(gu = tensor(args[0])) || !weight_of(args[1], &weight) || !silu_fits(*gu, weight)) Py_RETURN_NONE;
  refuse_tangent(*gu);
  if (weight) refuse_tangent(*weight);
  at::Tensor out;
  {
    Unlocked unlocked;
    out = at::GradMode::is_enabled() && (gu->requires_grad() || (weight && weight->requires_grad())) ? SiluMul::apply(*gu, weight)
                                                                                                    : silu(*gu, weight);
  }
  return THPVariable_Wrap(std::move(out));
  FMOE_CATCH
}

PyObject* py_silu_mul_quantise(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FMOE_TRY
  const at::Tensor* gu;
  std::optional<at::Tensor> weight;
  if (n != 3 || traced() || !(gu = tensor(args[0])) || !weight_of(args[2], &weight) || !silu_fits(*gu, weight) || gu->size(1) % 256 != 0)
    Py_RETURN_NONE;
  const bool hw = PyLong_AsLong(args[1]) == FMOE_QUANT_BLOCK128_UE8M0;
  const int64_t rows = gu->size(0), width = gu->size(1) / 2, groups = width / 128;
  const auto options = gu->options().dtype(at::kByte).requires_grad(false);
  at::Tensor q, scales;
  {
    Unlocked unlocked;
    q = at::empty({rows, width}, options);
    scales = at::empty({rows, hw ? (groups + 3) / 4 * 4 : 4 * groups}, options);
    check(F.silu_quantise(gu->data_ptr(), weight_ptr(weight), rows, static_cast<int32_t>(width), dtype_code(*gu),
                          hw ? FMOE_QUANT_BLOCK128_UE8M0 : FMOE_QUANT_BLOCK128, q.data_ptr(), scales.data_ptr(), stream_of(*gu)));
  }
  PyObject* both = PyTuple_New(2);
  if (both == nullptr) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(q));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(scales));
  return both;
  FMOE_CATCH
}

// For the backward of a node recorded in Python, on the current stream's device.
PyObject* py_check_capture(PyObject*, PyObject*) {
  FMOE_TRY
  refuse_default_stream_in_capture(c10::cuda::current_device());
  Py_RETURN_NONE;
  FMOE_CATCH
}

// bind(FmoeError, grouped_matmul, wgrad, block128, silu, silu_quantise, silu_backward, last_error): the
// class, then addresses.
PyObject* py_bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "an exception class and seven addresses");
    return nullptr;
  }
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i + 1]);
    if (p[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  Py_XDECREF(g_error_class);
  g_error_class = args[0];
  Py_INCREF(g_error_class);
  F.grouped = reinterpret_cast<decltype(F.grouped)>(p[0]);
  F.wgrad = reinterpret_cast<decltype(F.wgrad)>(p[1]);
  F.block128 = reinterpret_cast<decltype(F.block128)>(p[2]);
  F.silu = reinterpret_cast<decltype(F.silu)>(p[3]);
  F.silu_quantise = reinterpret_cast<decltype(F.silu_quantise)>(p[4]);
  F.silu_backward = reinterpret_cast<decltype(F.silu_backward)>(p[5]);
  F.last_error = reinterpret_cast<decltype(F.last_error)>(p[6]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef kMethods[] = {{"bind", FAST(py_bind), METH_FASTCALL, nullptr},
                          {"grouped_matmul", FAST(py_grouped_matmul), METH_FASTCALL, nullptr},
                          {"matmul_block128", FAST(py_matmul_block128), METH_FASTCALL, nullptr},
                          {"silu_mul", FAST(py_silu_mul), METH_FASTCALL, nullptr},
                          {"silu_mul_quantise", FAST(py_silu_mul_quantise), METH_FASTCALL, nullptr},
                          {"check_capture", py_check_capture, METH_NOARGS, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fmoe_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fmoe_torch() { return PyModule_Create(&kModule); }
