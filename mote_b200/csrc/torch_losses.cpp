// The losses' torch binding: checks tensors, allocates outputs and scratch through PyTorch's caching allocator and calls the
// C ABI (include/moteopt.h) on the current stream. A call of the losses is a few microseconds of device time on small inputs;
// the same checks, allocations and argument structures from Python took 12 to 29 us a call.
//
// The library is the one _lib.py has loaded: init() takes its functions' addresses.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "moteopt.h"

namespace {

struct Api {
  decltype(&moteopt_last_error) last_error;
  decltype(&moteopt_token_logprobs_workspace_size) logprobs_size;
  decltype(&moteopt_token_logprobs) token_logprobs;
  decltype(&moteopt_token_logprobs_backward) token_logprobs_backward;
  decltype(&moteopt_policy_loss_workspace_size) policy_size;
  decltype(&moteopt_policy_loss) policy;
  decltype(&moteopt_preference_loss_workspace_size) preference_size;
  decltype(&moteopt_preference_loss) preference;
} api;
PyObject* lib_error = nullptr;   // _lib.MoteoptError
PyObject* oom_error = nullptr;   // torch.OutOfMemoryError

constexpr size_t kHeader = 256;   // a workspace of no more than its header is not needed

struct Raised {};   // a Python error is set

[[noreturn]] void refuse(PyObject* kind, const std::string& why) {
  PyErr_SetString(kind, why.c_str());
  throw Raised();
}
std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t d : t.sizes()) s += (s.size() > 1 ? ", " : "") + std::to_string(d);
  return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(what) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.is_neg())   // its memory holds the values before the negation
    refuse(PyExc_ValueError, std::string(what) + " is a view that negates when it is read: resolve_neg() it");
  if (t._fw_grad(0).defined())
    refuse(PyExc_ValueError, std::string(what) + " carries a forward-mode tangent, which the losses do not have: detach() it");
  return t;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v != 0;
}

moteopt_logits logits_of(const at::Tensor& z) {
  int dtype = MOTEOPT_DTYPE_BF16;
  if (z.scalar_type() == at::kFloat) dtype = MOTEOPT_DTYPE_F32;
  else if (z.scalar_type() != at::kBFloat16)
    refuse(PyExc_TypeError, std::string("logits must be fp32 or bf16, got ") + c10::toString(z.scalar_type()));
  if (!z.is_cuda()) refuse(PyExc_ValueError, "logits must be a CUDA tensor (the losses run only on the GPU)");
  const int64_t n = z.dim();
  if (n != 2 && n != 3) refuse(PyExc_ValueError, "logits must be [S, T, V] or [N, V], got " + shape_of(z));
  const int64_t vocab = z.size(n - 1);
  if (vocab == 0) refuse(PyExc_ValueError, "logits have no vocabulary");
  if (z.stride(n - 1) != 1 && vocab > 1) refuse(PyExc_ValueError, "the logits' last axis must be contiguous");
  if (n == 3) return {z.data_ptr(), dtype, z.size(0), z.size(1), vocab, z.stride(0), z.stride(1)};
  return {z.data_ptr(), dtype, 1, z.size(0), vocab, 0, z.stride(0)};
}
moteopt_positions targets_of(const at::Tensor& y, const at::Tensor& z) {
  if (y.scalar_type() != at::kLong)
    refuse(PyExc_TypeError, std::string("targets must be int64, got ") + c10::toString(y.scalar_type()));
  if (y.sizes() != z.sizes().slice(0, z.dim() - 1))
    refuse(PyExc_ValueError, "targets " + shape_of(y) + " do not match logits " + shape_of(z));
  if (y.device() != z.device()) refuse(PyExc_ValueError, "targets must be on the logits' device");
  if (y.dim() == 2) return {y.data_ptr(), y.stride(0), y.stride(1)};
  return {y.data_ptr(), 0, y.stride(0)};
}
// fp32 values of the targets' shape, or [S] for [S, T] targets where `per_sequence`; none for None
moteopt_positions positions_of(PyObject* o, const at::Tensor& y, const char* what, bool per_sequence = false) {
  if (o == Py_None) return {nullptr, 0, 0};
  const at::Tensor& t = tensor(o, what);
  if (t.scalar_type() != at::kFloat)
    refuse(PyExc_TypeError, std::string(what) + " must be fp32, got " + c10::toString(t.scalar_type()));
  if (t.device() != y.device()) refuse(PyExc_ValueError, std::string(what) + " must be on the logits' device");
  if (t.sizes() == y.sizes()) {
    if (t.dim() == 2) return {t.data_ptr(), t.stride(0), t.stride(1)};
    return {t.data_ptr(), 0, t.stride(0)};
  }
  if (per_sequence && y.dim() == 2 && t.dim() == 1 && t.size(0) == y.size(0)) return {t.data_ptr(), t.stride(0), 0};
  refuse(PyExc_ValueError, std::string(what) + " " + shape_of(t) + " does not match targets " + shape_of(y));
}
const at::Tensor& required(PyObject* o, const char* what) {
  if (o == Py_None) refuse(PyExc_TypeError, std::string(what) + " must be a tensor, got None");
  return tensor(o, what);
}
const float* scalar_of(PyObject* o, const at::Tensor& z) {   // a divisor on the device, made so by the caller
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "divisor");
  if (t.scalar_type() != at::kFloat || t.numel() != 1 || t.device() != z.device())
    refuse(PyExc_ValueError, "divisor must be a one-element fp32 tensor on the logits' device");
  return t.const_data_ptr<float>();
}

// 0-dim tensor of a vector's element, on its storage (select() through the dispatcher takes half a microsecond each)
at::Tensor element(const at::Tensor& v, int64_t i) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(v.storage()), v.key_set(), v.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(v.storage_offset() + i);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({});
  return t;
}

// an uninitialised tensor on z's device, from PyTorch's caching allocator without the dispatcher
at::Tensor make(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& z) {
  return at::detail::empty_cuda(sizes, type, z.device(), std::nullopt);
}
at::Tensor scratch(size_t bytes, const at::Tensor& z) { return make({static_cast<int64_t>(bytes)}, at::kByte, z); }

moteopt_stream_t stream_of(const at::Tensor& z) {
  return reinterpret_cast<moteopt_stream_t>(c10::cuda::getCurrentCUDAStream(z.get_device()).stream());
}
PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* tuple(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!r) throw Raised();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = nullptr;
    if (t.defined()) o = wrap(t);
    else Py_INCREF(o = Py_None);
    if (!o) {
      Py_DECREF(r);
      throw Raised();
    }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

// Other Python threads run while a call allocates and launches: it waits where the launch queue is full, on work that may itself
// wait for one of them (a host function in a stream), or for memory.
struct Threads {
  PyThreadState* const state = PyEval_SaveThread();
  ~Threads() { PyEval_RestoreThread(state); }
};

// `call` allocates and launches, the logits' device current; an error of the library is Python's
template <typename F>
void checked(const char* what, const at::Tensor& z, F call) {
  int rc;
  std::string why;
  {
    const Threads others;
    const c10::cuda::CUDAGuard guard(z.device());
    rc = call();
    if (rc != MOTEOPT_OK) why = api.last_error();   // of this thread
  }
  if (rc != MOTEOPT_OK) refuse(lib_error, std::string(what) + " failed (" + std::to_string(rc) + "): " + why);
}

// An entry point: nothing recorded for autograd, C++ errors as Python's
template <typename F>
PyObject* entry(Py_ssize_t given, Py_ssize_t wanted, F body) {
  if (given != wanted) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
    return nullptr;
  }
  try {
    c10::impl::ExcludeDispatchKeyGuard no_autograd(c10::autograd_dispatch_keyset);
    return body();
  } catch (const Raised&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(oom_error, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (logits, targets, temperature) -> (logprobs, lse)
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 3, [&] {
    const at::Tensor &z = required(a[0], "logits"), &y = required(a[1], "targets");
    const moteopt_logits L = logits_of(z);
    const moteopt_positions Y = targets_of(y, z);
    const double t = number(a[2]);
    at::Tensor logp, lse;
    checked("moteopt_token_logprobs", z, [&] {
      logp = make(y.sizes(), at::kFloat, z);
      lse = make(y.sizes(), at::kFloat, z);
      const size_t bytes = api.logprobs_size(&L);
      at::Tensor ws;
      if (bytes > kHeader) ws = scratch(bytes, z);
      return api.token_logprobs(&L, &Y, t, logp.data_ptr<float>(), lse.data_ptr<float>(),
                                ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? bytes : 0, stream_of(z));
    });
    return tuple({logp, lse});
  });
}

// (logits, targets, logprobs, lse, grad_logprobs, temperature) -> grad
PyObject* token_logprobs_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 6, [&] {
    const at::Tensor &z = required(a[0], "logits"), &y = required(a[1], "targets");
    const moteopt_logits L = logits_of(z);
    const moteopt_positions Y = targets_of(y, z);
    for (int k = 2; k < 5; ++k) required(a[k], k == 2 ? "logprobs" : k == 3 ? "lse" : "grad_logprobs");
    const moteopt_positions P = positions_of(a[2], y, "logprobs"), S = positions_of(a[3], y, "lse");
    const moteopt_positions G = positions_of(a[4], y, "grad_logprobs", true);
    const double t = number(a[5]);
    at::Tensor grad;
    checked("moteopt_token_logprobs_backward", z, [&] {
      grad = make(z.sizes(), z.scalar_type(), z);
      return api.token_logprobs_backward(&L, &Y, t, &P, &S, &G, grad.data_ptr(), stream_of(z));
    });
    return wrap(grad);
  });
}

// (logits, targets, advantages, old_logprobs, ref_logprobs | None, weights | None, clip_low, clip_high, kl_coef, temperature,
//  divisor, divisor on the device | None, grad) -> (loss, count, kl, clipped, logprobs, grad | None)
PyObject* policy_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 13, [&] {
    const at::Tensor &z = required(a[0], "logits"), &y = required(a[1], "targets");
    const moteopt_logits L = logits_of(z);
    const moteopt_positions Y = targets_of(y, z);
    required(a[2], "advantages");
    required(a[3], "old_logprobs");
    moteopt_policy P;
    P.advantages = positions_of(a[2], y, "advantages", true);
    P.old_logprobs = positions_of(a[3], y, "old_logprobs");
    P.ref_logprobs = positions_of(a[4], y, "ref_logprobs");
    P.weights = positions_of(a[5], y, "weights", true);
    P.clip_low = number(a[6]);
    P.clip_high = number(a[7]);
    P.kl_coef = number(a[8]);
    const double t = number(a[9]);
    P.divisor = number(a[10]);
    P.divisor_device = scalar_of(a[11], z);
    const bool with_grad = truth(a[12]);
    if (P.kl_coef != 0.0 && a[4] == Py_None) refuse(PyExc_ValueError, "policy_loss: kl_coef needs ref_logprobs");
    at::Tensor sums, logp, grad;
    checked("moteopt_policy_loss", z, [&] {
      const size_t bytes = api.policy_size(&L);
      const at::Tensor ws = scratch(bytes, z);
      sums = make({4}, at::kFloat, z);
      logp = make(y.sizes(), at::kFloat, z);
      if (with_grad) grad = make(z.sizes(), z.scalar_type(), z);
      return api.policy(&L, &Y, &P, t, sums.data_ptr<float>(), logp.data_ptr<float>(), with_grad ? grad.data_ptr() : nullptr,
                        ws.data_ptr(), bytes, stream_of(z));
    });
    return tuple({element(sums, 0), element(sums, 1), element(sums, 2), element(sums, 3), logp, grad});
  });
}

// (logits, targets, ref_logprobs | None, cu_seqlens | None, beta, label_smoothing, average, temperature, divisor, divisor on
//  the device | None, grad) -> (loss, rewards, logprobs, grad | None)
PyObject* preference_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return entry(n, 11, [&] {
    const at::Tensor &z = required(a[0], "logits"), &y = required(a[1], "targets");
    const moteopt_logits L = logits_of(z);
    const moteopt_positions Y = targets_of(y, z);
    moteopt_preference P = {};
    if (a[3] != Py_None) {
      const at::Tensor& cu = tensor(a[3], "cu_seqlens");
      if (z.dim() != 2) refuse(PyExc_ValueError, "preference_loss: cu_seqlens goes with [N, V] logits");
      if (cu.scalar_type() != at::kInt || cu.dim() != 1 || !cu.is_contiguous())
        refuse(PyExc_TypeError, "cu_seqlens must be a contiguous int32 vector");
      if (cu.device() != z.device()) refuse(PyExc_ValueError, "cu_seqlens must be on the logits' device");
      P.cu_seqlens = cu.const_data_ptr<int32_t>();
      P.sequences = cu.numel() - 1;
    } else {
      if (z.dim() != 3) refuse(PyExc_ValueError, "preference_loss: [N, V] logits need cu_seqlens");
      P.sequences = z.size(0);
    }
    if (P.sequences < 0 || P.sequences % 2)
      refuse(PyExc_ValueError, "preference_loss: chosen and rejected sequences come in pairs, got " + std::to_string(P.sequences));
    if (a[2] != Py_None) {
      const at::Tensor& ref = tensor(a[2], "ref_logprobs");
      if (ref.scalar_type() != at::kFloat)
        refuse(PyExc_TypeError, std::string("ref_logprobs must be fp32, got ") + c10::toString(ref.scalar_type()));
      if (ref.dim() != 1 || ref.size(0) != P.sequences || ref.device() != z.device() || !ref.is_contiguous())
        refuse(PyExc_ValueError, "ref_logprobs must be a contiguous vector of " + std::to_string(P.sequences) +
                                     " on the logits' device");
      P.ref_logprobs = ref.const_data_ptr<float>();
    }
    P.beta = number(a[4]);
    P.label_smoothing = number(a[5]);
    P.average = truth(a[6]);
    const double t = number(a[7]);
    P.divisor = number(a[8]);
    P.divisor_device = scalar_of(a[9], z);
    const bool with_grad = truth(a[10]);
    at::Tensor loss, rewards, logp, grad;
    checked("moteopt_preference_loss", z, [&] {
      const size_t bytes = api.preference_size(&L, P.sequences);
      const at::Tensor ws = scratch(bytes, z);
      loss = make({}, at::kFloat, z);
      rewards = make({P.sequences}, at::kFloat, z);
      logp = make({P.sequences}, at::kFloat, z);
      if (with_grad) grad = make(z.sizes(), z.scalar_type(), z);
      return api.preference(&L, &Y, &P, t, loss.data_ptr<float>(), rewards.data_ptr<float>(), logp.data_ptr<float>(),
                            with_grad ? grad.data_ptr() : nullptr, ws.data_ptr(), bytes, stream_of(z));
    });
    return tuple({loss, rewards, logp, grad});
  });
}

// init(addresses of the functions in Api's order, MoteoptError, torch.OutOfMemoryError)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void** const slots = reinterpret_cast<void**>(&api);
  constexpr Py_ssize_t kFns = sizeof(Api) / sizeof(void*);
  if (n != kFns + 2) {
    PyErr_SetString(PyExc_TypeError, "init: wrong number of arguments");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < kFns; ++i) {
    slots[i] = PyLong_AsVoidPtr(a[i]);
    if (slots[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "init: null function");
      return nullptr;
    }
  }
  Py_INCREF(a[kFns]);
  Py_XSETREF(lib_error, a[kFns]);
  Py_INCREF(a[kFns + 1]);
  Py_XSETREF(oom_error, a[kFns + 1]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}
PyMethodDef methods[] = {{"init", fast<init>(), METH_FASTCALL, nullptr},
                         {"token_logprobs", fast<token_logprobs>(), METH_FASTCALL, nullptr},
                         {"token_logprobs_backward", fast<token_logprobs_backward>(), METH_FASTCALL, nullptr},
                         {"policy_loss", fast<policy_loss>(), METH_FASTCALL, nullptr},
                         {"preference_loss", fast<preference_loss>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
// looked for by build.py before the binding is loaded
constexpr const char* kDoc = "The losses' torch binding, built for " MOTEOPT_BUILT_FOR ".";
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_losses", kDoc, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_losses(void) { return PyModule_Create(&module); }
