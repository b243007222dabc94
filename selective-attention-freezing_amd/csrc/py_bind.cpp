// CPython module kernel._bind: the host path of the decoding and training operators where
// ctypes and Python cost more than the kernels.
//
// fill(what, block, offsets, rows, device, refuse_grad, t0, t1, ...) writes the
// saf_tensor_t of each tensor (None: left as it is) at block + offsets[i].
// It raises where a tensor is not on HIP device `device`, has more than four
// dimensions or a dtype the library does not know, carries a forward-mode
// tangent, or (refuse_grad) needs a gradient while grad mode is on.  Bit i of `rows` asks for rows of tensor i
// (4-D, only read) to be 16-byte aligned with a unit last stride; the result
// has the bits of those that are not.
//
// The same through ctypes costs about 0.6 us a tensor, half of the host time
// of a single-token call; here the tensor's fields are read directly.
//
// token_logprobs(logits, tokens, top, entropy, scale, ignore_index) runs
// saf_token_logprobs on (R, V) logits and (R,) tokens and returns (logp, entropy
// or None, top_index or None, top_logp or None), differentiable in the logits.
// As an autograd node in C++ its backward runs in the engine's thread without
// the interpreter: forward and backward of a small call took 90-110 us as a
// Python autograd.Function.
//
// embed_tokens, add_layernorm, gelu_packed and their like are in
// py_bind_train.cpp.
//
// library(addresses) hands over the entry points of libsafattn.so.
#include "py_bind.h"

using namespace saf_bind;

namespace saf_bind {

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SAF_F32;
    case at::kHalf: return SAF_F16;
    case at::kBFloat16: return SAF_BF16;
    case at::kInt: return SAF_I32;
    case at::kLong: return SAF_I64;
    default: return -1;
  }
}

static decltype(&saf_last_error) last_error = nullptr;

bool has_tangent(const at::Tensor& x) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined();
}

void check(int rc) {
  if (rc == SAF_OK) return;
  TORCH_CHECK_NOT_IMPLEMENTED(rc != SAF_EUNSUPPORTED, last_error());
  TORCH_CHECK_VALUE(rc != SAF_EINVAL && rc != SAF_EALIGN && rc != SAF_EWORKSPACE, last_error());
  TORCH_CHECK(false, last_error());
}

// dimensions that a descriptor has room for
constexpr int kMaxDims = sizeof(saf_tensor_t::size) / sizeof(int64_t);

saf_tensor_t desc(const char* what, const at::Tensor& x) {
  saf_tensor_t d{};
  if (!x.defined()) return d;
  const int code = dtype_code(x.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(code >= 0, what, ": unsupported dtype ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() <= kMaxDims, what, ": tensors have at most ", kMaxDims, " dimensions");
  d.data = x.data_ptr();
  d.dtype = code;
  d.ndim = (int32_t)x.dim();
  for (int k = 0; k < d.ndim; ++k) {
    d.size[k] = x.size(k);
    d.stride[k] = x.stride(k);
  }
  return d;
}

at::Tensor only_once(const char* what, at::Tensor dx) {
  if (!dx.defined() || !at::GradMode::is_enabled()) return dx;
  auto once = std::make_shared<torch::autograd::DelayedError>(std::string(what) + ": twice differentiating is not supported", 1);
  return (*once)({dx.detach().set_requires_grad(true)})[0];
}

void refuse_foreign_capture(const char* what, const char* name, const at::Tensor& x) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> leaves;
  if (auto fn = x.grad_fn()) {
    for (;;) {
      std::shared_ptr<torch::autograd::Node> only;
      int n = 0;
      for (const auto& e : fn->next_edges())
        if (e.function) {
          only = e.function;
          ++n;
        }
      if (n != 1 || only->num_outputs() == 0) break;  // the leaf's own node has no next edges
      fn = std::move(only);
    }
    for (const auto& e : fn->next_edges())
      if (e.function && e.function->name() == "torch::autograd::AccumulateGrad") leaves.push_back(e.function);
  } else if (auto node = torch::autograd::impl::try_get_grad_accumulator(x)) {
    leaves.push_back(std::move(node));
  }
  const c10::Stream now = c10::hip::getCurrentHIPStream().unwrap();
  for (const auto& node : leaves) {
    const auto made = node->stream();
    TORCH_CHECK(!made || made->id() == now.id(),
                what, ": an eager autograd graph of these ", name, ", made on another stream, is still alive; release "
                "it before capturing their gradient");
  }
}

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

}  // namespace saf_bind

namespace {

bool rows_ok(const at::Tensor& x) {
  if (x.dim() != 4) return true;  // the library names the mistake
  const int64_t es = x.element_size();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || (x.size(3) > 1 && x.stride(3) != 1)) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size(i) > 1 && x.stride(i) * es % 16) return false;
  return true;
}

PyObject* fill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t kFixed = 6;
  if (n < kFixed || !PyTuple_Check(args[2]) || PyTuple_GET_SIZE(args[2]) != n - kFixed) {
    PyErr_SetString(PyExc_TypeError, "fill(what, block, offsets, rows, device, refuse_grad, *tensors)");
    return nullptr;
  }
  const char* what = PyUnicode_AsUTF8(args[0]);
  char* block = static_cast<char*>(PyLong_AsVoidPtr(args[1]));
  const long rows = PyLong_AsLong(args[3]), device = PyLong_AsLong(args[4]);
  const int refuse = PyObject_IsTrue(args[5]);
  if (what == nullptr || PyErr_Occurred()) return nullptr;
  long copies = 0;
  for (Py_ssize_t i = 0; i < n - kFixed; ++i) {
    PyObject* o = args[kFixed + i];
    if (o == Py_None) continue;
    if (!THPVariable_Check(o)) return PyErr_Format(PyExc_TypeError, "%s: a tensor is required, got %R", what, Py_TYPE(o));
    const at::Tensor& x = THPVariable_Unpack(o);
    if (has_tangent(x)) return PyErr_Format(PyExc_NotImplementedError, "%s has no forward-mode derivative", what);
    if (!x.is_cuda() || x.device().index() != device)
      return PyErr_Format(PyExc_ValueError, "%s: a tensor is on %s, expected cuda:%ld", what, x.device().str().c_str(),
                          device);
    if (refuse && x.requires_grad() && at::GradMode::is_enabled())
      return PyErr_Format(PyExc_NotImplementedError, "%s has no backward: call it under torch.no_grad()", what);
    const int code = dtype_code(x.scalar_type());
    if (code < 0)
      return PyErr_Format(PyExc_NotImplementedError, "%s: unsupported dtype %s", what, c10::toString(x.scalar_type()));
    if (x.dim() > kMaxDims) return PyErr_Format(PyExc_ValueError, "%s: tensors have at most %d dimensions", what, kMaxDims);
    if (rows >> i & 1 && !rows_ok(x)) {
      copies |= 1L << i;
      continue;
    }
    saf_tensor_t* d = reinterpret_cast<saf_tensor_t*>(block + PyLong_AsLong(PyTuple_GET_ITEM(args[2], i)));
    *d = saf_tensor_t{};
    d->data = x.data_ptr();
    d->dtype = code;
    d->ndim = (int32_t)x.dim();
    for (int k = 0; k < d->ndim; ++k) {
      d->size[k] = x.size(k);
      d->stride[k] = x.stride(k);
    }
  }
  return PyLong_FromLong(copies);
}

PyObject* fill_checked(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return fill(self, args, n);
  END_HANDLE_TH_ERRORS
}

// ---- token_logprobs --------------------------------------------------------------

struct {
  decltype(&saf_token_logprobs) forward;
  decltype(&saf_token_logprobs_workspace_bytes) workspace_bytes;
  decltype(&saf_token_logprobs_bwd) backward;
} lib{};

constexpr const char* kWhat = "token_logprobs";

struct Options {
  int64_t top, ignore;
  bool entropy;
  double scale;
};
struct Outputs {
  at::Tensor logp, entropy, index, top_logp, stats;
};

saf_token_logprobs_args arguments(const at::Tensor& logits, const at::Tensor& tokens, int64_t ignore, double scale) {
  saf_token_logprobs_args a{};
  a.logits = desc(kWhat, logits);
  a.tokens = desc(kWhat, tokens);
  a.ignore_index = ignore;
  a.scale = (float)scale;
  return a;
}

Outputs run_forward(const at::Tensor& logits, const at::Tensor& tokens, const Options& o, bool keep_stats) {
  const c10::hip::HIPGuard guard(logits.get_device());
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  const int64_t R = logits.size(0);
  Outputs r;
  r.logp = at::empty({R}, f32);
  if (o.entropy) r.entropy = at::empty({R}, f32);
  if (keep_stats) r.stats = at::empty({R, 2}, f32);
  if (o.top > 0) {
    r.index = at::empty({R, o.top}, f32.dtype(at::kLong));
    r.top_logp = at::empty({R, o.top}, f32);
  }
  saf_token_logprobs_args a = arguments(logits, tokens, o.ignore, o.scale);
  a.top = (int32_t)o.top;
  a.logp = desc(kWhat, r.logp);
  a.entropy = desc(kWhat, r.entropy);
  a.stats = desc(kWhat, r.stats);
  a.top_index = desc(kWhat, r.index);
  a.top_logp = desc(kWhat, r.top_logp);
  at::Tensor ws;
  const int64_t bytes = lib.workspace_bytes(&a);
  if (bytes > 0) {
    ws = at::empty({bytes}, f32.dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = bytes;
  }
  check(lib.forward(&a, c10::hip::getCurrentHIPStream().stream()));
  return r;
}

struct TokenLogprobs : public torch::autograd::Function<TokenLogprobs> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits,
                                                const at::Tensor& tokens, const Options& o) {
    Outputs r = run_forward(logits, tokens, o, true);
    ctx->save_for_backward({logits, tokens, r.stats, r.entropy});
    ctx->saved_data["scale"] = o.scale;
    ctx->saved_data["ignore"] = o.ignore;
    ctx->saved_data["entropy"] = o.entropy;
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list out{r.logp};
    if (o.entropy) out.push_back(r.entropy);
    if (o.top > 0) {
      out.push_back(r.index);
      out.push_back(r.top_logp);
      ctx->mark_non_differentiable({r.index, r.top_logp});
    }
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &tokens = saved[1], &stats = saved[2], &entropy = saved[3];
    const bool ent = ctx->saved_data["entropy"].toBool() && grads[1].defined();
    if (!grads[0].defined() && !ent) return {at::Tensor(), at::Tensor(), at::Tensor()};
    const c10::hip::HIPGuard guard(logits.get_device());
    at::Tensor dx;
    {
      at::NoGradGuard no_grad;
      const at::Tensor g = grads[0].defined() ? grads[0].to(at::kFloat)
                                              : at::zeros({logits.size(0)}, stats.options());
      const at::Tensor ge = ent ? grads[1].to(at::kFloat) : at::Tensor();
      dx = at::empty({logits.size(0), logits.size(1)}, logits.options().requires_grad(false));
      saf_token_logprobs_args a =
          arguments(logits, tokens, ctx->saved_data["ignore"].toInt(), ctx->saved_data["scale"].toDouble());
      a.stats = desc(kWhat, stats);
      a.entropy = desc(kWhat, entropy);
      const saf_tensor_t dg = desc(kWhat, g), dge = desc(kWhat, ge), ddx = desc(kWhat, dx);
      check(lib.backward(&a, &dg, &dge, &ddx, c10::hip::getCurrentHIPStream().stream()));
    }
    dx = only_once("token_logprobs", dx);
    return {dx, at::Tensor(), at::Tensor()};
  }
};

PyObject* token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "token_logprobs(logits, tokens, top, entropy, scale, ignore_index)");
    return nullptr;
  }
  TORCH_CHECK(lib.forward != nullptr, "libsafattn.so is not loaded");
  const at::Tensor &logits = THPVariable_Unpack(args[0]), &tokens = THPVariable_Unpack(args[1]);
  Options o{PyLong_AsLongLong(args[2]), PyLong_AsLongLong(args[5]), PyObject_IsTrue(args[3]) == 1, PyFloat_AsDouble(args[4])};
  if (PyErr_Occurred()) return nullptr;
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(logits), "token_logprobs has no forward-mode derivative");
  TORCH_CHECK_VALUE(logits.is_cuda() && tokens.device() == logits.device(), "token_logprobs: a tensor is on ",
                    tokens.device(), ", expected ", logits.device());
  TORCH_CHECK_NOT_IMPLEMENTED(o.top >= 0 && o.top <= 32, "top = ", o.top, " outside 0..32 or above the vocabulary");
  Outputs r;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    refuse_foreign_capture("token_logprobs", "logits", logits);
    const auto out = TokenLogprobs::apply(logits, tokens, o);
    size_t k = 0;
    r.logp = out[k++];
    if (o.entropy) r.entropy = out[k++];
    if (o.top > 0) {
      r.index = out[k++];
      r.top_logp = out[k++];
    }
  } else {
    r = run_forward(logits, tokens, o, false);
  }
  PyObject* t = PyTuple_New(4);
  if (t == nullptr) return nullptr;
  const at::Tensor* parts[4] = {&r.logp, &r.entropy, &r.index, &r.top_logp};
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(t, i, wrap(*parts[i]));
  return t;
  END_HANDLE_TH_ERRORS
}

PyObject* library(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "library(forward, workspace_bytes, backward, last_error)");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  lib.forward = reinterpret_cast<decltype(lib.forward)>(p[0]);
  lib.workspace_bytes = reinterpret_cast<decltype(lib.workspace_bytes)>(p[1]);
  lib.backward = reinterpret_cast<decltype(lib.backward)>(p[2]);
  last_error = reinterpret_cast<decltype(last_error)>(p[3]);
  Py_RETURN_NONE;
}

typedef PyObject* (*FastCall)(PyObject*, PyObject* const*, Py_ssize_t);
PyCFunction method(FastCall f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"fill", method(fill_checked), METH_FASTCALL,
     "fill(what, block, offsets, rows, device, refuse_grad, *tensors) -> mask of tensors whose rows need a copy"},
    {"token_logprobs", method(token_logprobs), METH_FASTCALL,
     "token_logprobs(logits, tokens, top, entropy, scale, ignore_index) -> (logp, entropy, top_index, top_logp)"},
    {"embed_tokens", method(embed_tokens), METH_FASTCALL, "embed_tokens(tokens, weight, scale, ignore_index, dtype) -> rows"},
    {"add_layernorm", method(add_layernorm), METH_FASTCALL,
     "add_layernorm(x, delta, weight, bias, eps, dtype) -> (r or None, y)"},
    {"gelu_packed", method(gelu_packed), METH_FASTCALL, "gelu_packed(x, keep) -> y, or (y, q, exp) with keep"},
    {"gelu_packed_bwd", method(gelu_packed_bwd), METH_FASTCALL, "gelu_packed_bwd(q, exp, dy, again) -> (dx, y or None)"},
    {"pack_activation", method(pack_activation), METH_FASTCALL, "pack_activation(x) -> (q, exp)"},
    {"unpack_activation", method(unpack_activation), METH_FASTCALL, "unpack_activation(q, exp, dtype) -> x"},
    {"check_differentiable", method(check_differentiable), METH_FASTCALL, "check_differentiable(what, *tensors)"},
    {"library_train", method(library_train), METH_FASTCALL, "library_train(addresses of the training operators)"},
    {"library", method(library), METH_FASTCALL, "library(forward, workspace_bytes, backward, last_error)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Host path of the decoding and training operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
