// The host path of the training operators in the CPython module kernel._bind:
//
// embed_tokens(tokens, weight, scale, ignore_index, dtype) -> rows
// add_layernorm(x, delta, weight, bias, eps, dtype) -> (r or None, y)
// gelu_packed(x, keep) -> y, or (y, q, exp) with keep
//     differentiable in weight; x, delta, weight and bias; x (without keep)
// gelu_packed_bwd(q, exp, dy, again) -> (dx, y or None)
// pack_activation(x) -> (q, exp), unpack_activation(q, exp, dtype) -> x
// check_differentiable(what, *tensors): the checks of the above for an operator
//     whose autograd node is Python's
//
// dtype is a code of the C-ABI, -1 for the operator's default.  The autograd nodes
// are C++, so that a backward pass takes neither the interpreter nor its lock.
// library_train(addresses) hands over the entry points of libsafattn.so.
#include "py_bind.h"

#include <ATen/ops/empty_like.h>

#include <optional>

namespace saf_bind {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct {
  decltype(&saf_embed_fwd) embed;
  decltype(&saf_embed_bwd) embed_bwd;
  decltype(&saf_embed_bwd_workspace_bytes) embed_bytes;
  decltype(&saf_layernorm_fwd) layernorm;
  decltype(&saf_layernorm_bwd) layernorm_bwd;
  decltype(&saf_layernorm_bwd_workspace_bytes) layernorm_bytes;
  decltype(&saf_act_pack) pack;
  decltype(&saf_act_unpack) unpack;
  decltype(&saf_gelu_pack_fwd) gelu;
  decltype(&saf_gelu_pack_bwd) gelu_bwd;
} lib{};

at::ScalarType type_of(long code, at::ScalarType otherwise) {
  switch (code) {
    case SAF_F32: return at::kFloat;
    case SAF_F16: return at::kHalf;
    case SAF_BF16: return at::kBFloat16;
    default: return otherwise;
  }
}

void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

at::TensorOptions plain(const at::Tensor& x) { return x.options().requires_grad(false); }

// (..., C) as rows (R, C) with a unit column stride: a view where it can be one.
at::Tensor rows(const at::Tensor& x) {
  at::Tensor t = x;
  if (t.dim() != 2) {
    const int64_t C = t.size(-1);
    int64_t R = 1;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) R *= t.size(i);
    t = t.reshape({R, C});
  }
  return t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t;
}

// Descriptor of (..., C) rows that rows() returned or a new contiguous tensor.
saf_tensor_t rows_desc(const char* what, const at::Tensor& x) {
  saf_tensor_t d{};
  if (!x.defined()) return d;
  d.data = x.data_ptr();
  d.dtype = x.scalar_type() == at::kChar ? SAF_I8 : x.scalar_type() == at::kByte ? SAF_U8 : dtype_code(x.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(d.dtype >= 0, what, ": unsupported dtype ", x.scalar_type());
  const int64_t C = x.size(-1);
  int64_t R = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) R *= x.size(i);
  d.ndim = 2;
  d.size[0] = R;
  d.size[1] = C;
  d.stride[0] = x.dim() == 2 ? x.stride(0) : C;
  d.stride[1] = 1;
  return d;
}

// A (C,) vector with a unit stride.
at::Tensor vec(const at::Tensor& x) { return x.defined() && x.dim() == 1 && x.size(0) > 1 && x.stride(0) != 1 ? x.contiguous() : x; }

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, plain(like).dtype(at::kByte)) : at::Tensor();
}
void* data(const at::Tensor& x) { return x.defined() ? x.data_ptr() : nullptr; }

// A tensor argument on a HIP device, without a tangent.
const at::Tensor& tensor(const char* what, PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": a tensor is required");
  const at::Tensor& x = THPVariable_Unpack(o);
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(x), what, " has no forward-mode derivative");
  return x;
}
void same_device(const char* what, const at::Tensor& x, const at::Tensor& as) {
  TORCH_CHECK(as.is_cuda(), what, " runs on HIP devices only (got a CPU tensor)");
  TORCH_CHECK_VALUE(x.device() == as.device(), what, ": a tensor is on ", x.device(), ", expected ", as.device());
}
void check_vector(const char* what, const char* name, const at::Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 1, what, ": ", name, " must be a (C,) vector (got ", x.sizes(), ")");
}
bool recorded(const at::Tensor& x) { return x.defined() && x.requires_grad() && at::GradMode::is_enabled(); }

// ---- embed_tokens ----------------------------------------------------------------

constexpr const char* kEmbed = "embed_tokens";

struct EmbedOptions {
  double scale;
  int64_t ignore;
  at::ScalarType type;
};

at::Tensor embed_forward(const at::Tensor& tokens, const at::Tensor& weight, const EmbedOptions& o) {
  const c10::hip::HIPGuard guard(weight.get_device());
  auto sizes = tokens.sizes().vec();
  sizes.push_back(weight.size(1));
  at::Tensor y = at::empty(sizes, plain(weight).dtype(o.type));
  const at::Tensor t = tokens.dim() == 1 ? tokens : tokens.reshape({tokens.numel()}), w = rows(weight);
  const saf_tensor_t td = desc(kEmbed, t), wd = rows_desc(kEmbed, w), yd = rows_desc(kEmbed, y);
  check(lib.embed(&td, &wd, (float)o.scale, o.ignore, &yd, stream()));
  return y;
}

struct EmbedTokens : public torch::autograd::Function<EmbedTokens> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& weight, const at::Tensor& tokens,
                               const EmbedOptions& o) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["scale"] = o.scale;
    ctx->saved_data["ignore"] = o.ignore;
    ctx->saved_data["V"] = weight.size(0);
    ctx->saved_data["type"] = (int64_t)weight.scalar_type();
    ctx->set_materialize_grads(false);
    return {embed_forward(tokens, weight, o)};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    const at::Tensor tokens = ctx->get_saved_variables()[0];
    const c10::hip::HIPGuard guard(grads[0].get_device());
    at::Tensor dw;
    {
      at::NoGradGuard no_grad;
      const at::Tensor g = rows(grads[0]), t = tokens.dim() == 1 ? tokens : tokens.reshape({tokens.numel()});
      const int64_t V = ctx->saved_data["V"].toInt(), C = g.size(1);
      dw = at::empty({V, C}, plain(g).dtype((at::ScalarType)ctx->saved_data["type"].toInt()));
      const int64_t bytes = lib.embed_bytes(t.numel(), V, C);
      if (bytes < 0) check(SAF_EUNSUPPORTED);
      const at::Tensor ws = workspace(bytes, g);
      const saf_tensor_t td = desc(kEmbed, t), gd = rows_desc(kEmbed, g), dd = rows_desc(kEmbed, dw);
      check(lib.embed_bwd(&td, &gd, (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["ignore"].toInt(), &dd,
                          data(ws), bytes, stream()));
    }
    return {only_once(kEmbed, dw), at::Tensor(), at::Tensor()};
  }
};

// ---- add_layernorm ----------------------------------------------------------------

constexpr const char* kNorm = "add_layernorm";

struct NormOptions {
  double eps;
  at::ScalarType type;
};
struct NormOutputs {
  at::Tensor r, y, stats;
};

NormOutputs norm_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& delta, const at::Tensor& bias,
                         const NormOptions& o, bool keep) {
  const c10::hip::HIPGuard guard(x.get_device());
  NormOutputs n;
  const at::Tensor x2 = rows(x), w = vec(weight), b = vec(bias);
  at::Tensor d2;
  if (delta.defined()) {
    d2 = rows(delta);
    n.r = at::empty(x.sizes(), plain(x));
  }
  n.y = at::empty(x.sizes(), plain(x).dtype(o.type));
  const saf_tensor_t xd = rows_desc(kNorm, x2);
  if (keep) n.stats = at::empty({xd.size[0], 2}, plain(x).dtype(at::kFloat));
  const saf_tensor_t dd = rows_desc(kNorm, d2), wd = desc(kNorm, w), bd = desc(kNorm, b), rd = rows_desc(kNorm, n.r),
                     yd = rows_desc(kNorm, n.y), sd = rows_desc(kNorm, n.stats);
  check(lib.layernorm(&xd, &dd, &wd, &bd, (float)o.eps, &rd, &yd, &sd, stream()));
  return n;
}

struct AddLayernorm : public torch::autograd::Function<AddLayernorm> {
  // gradients of the inputs in the order x, weight, delta (where there is one), bias
  // (where there is one): absent optionals are no inputs of the node
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight,
                               const std::optional<at::Tensor>& delta, const std::optional<at::Tensor>& bias,
                               const NormOptions& o) {
    const NormOutputs n = norm_forward(x, weight, delta ? *delta : at::Tensor(), bias ? *bias : at::Tensor(), o, true);
    ctx->save_for_backward({n.r.defined() ? n.r : x, weight, n.stats});
    ctx->saved_data["delta"] = delta.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["branch"] = (int64_t)o.type;
    ctx->set_materialize_grads(false);
    if (n.r.defined()) return {n.r, n.y};
    return {n.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool has_d = ctx->saved_data["delta"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    at::Tensor dr = has_d ? grads[0] : at::Tensor(), dy = grads[has_d ? 1 : 0];
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1),
               want_d = has_d && ctx->needs_input_grad(2), want_b = has_b && ctx->needs_input_grad(has_d ? 3 : 2);
    at::Tensor dx, dw, dd, db;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &r = saved[0], &weight = saved[1], &stats = saved[2];
    if (dy.defined() && (want_x || want_w || want_d || want_b)) {
      const c10::hip::HIPGuard guard(r.get_device());
      at::NoGradGuard no_grad;
      const at::Tensor r2 = rows(r), g2 = rows(dy), w = vec(weight);
      at::Tensor e2;
      if (dr.defined()) e2 = rows(dr);
      // one tensor serves both gradients of a sum of one type
      const bool same = r.scalar_type() == dy.scalar_type();
      if (want_x || (want_d && same)) dx = at::empty(r.sizes(), plain(r));
      if (want_d) dd = same ? dx : at::empty(r.sizes(), plain(dy));
      if (want_w) dw = at::empty(weight.sizes(), plain(weight));
      if (want_b) db = at::empty(weight.sizes(), plain(weight));
      const saf_tensor_t rd = rows_desc(kNorm, r2), sd = rows_desc(kNorm, stats), wd = desc(kNorm, w),
                         gd = rows_desc(kNorm, g2), ed = rows_desc(kNorm, e2), xd = rows_desc(kNorm, dx),
                         ddd = rows_desc(kNorm, same ? at::Tensor() : dd), dwd = desc(kNorm, dw), dbd = desc(kNorm, db);
      int64_t bytes = 0;
      if (want_w || want_b) {
        bytes = lib.layernorm_bytes(rd.size[0], rd.size[1]);
        if (bytes < 0) check(SAF_EINVAL);
      }
      const at::Tensor ws = workspace(bytes, r);
      check(lib.layernorm_bwd(&rd, &sd, &wd, &gd, &ed, &xd, &ddd, &dwd, &dbd, data(ws), bytes, stream()));
      if (!want_x) dx = at::Tensor();
    } else if (dr.defined()) {  // y has no part in it: the sum's own gradient
      if (want_x) dx = dr;
      if (want_d) dd = dr.to((at::ScalarType)ctx->saved_data["branch"].toInt());
    }
    variable_list out{only_once(kNorm, dx), only_once(kNorm, dw), at::Tensor(), at::Tensor(), at::Tensor()};
    if (want_d) out[2] = dd.is_same(dx) ? out[0] : only_once(kNorm, dd);
    if (want_b) out[3] = only_once(kNorm, db);
    return out;
  }
};

// ---- 8-bit activations --------------------------------------------------------------

constexpr const char* kGelu = "gelu_packed";

struct Packed {
  at::Tensor q, exp;
};
void check_channels(const at::Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "an activation has at least one channel");
}
Packed packed_like(const at::Tensor& x) {
  auto sizes = x.sizes().vec();
  sizes.back() = (sizes.back() + 31) / 32;
  return {at::empty(x.sizes(), plain(x).dtype(at::kChar)), at::empty(sizes, plain(x).dtype(at::kByte))};
}

struct GeluOutputs {
  at::Tensor y;
  Packed p;
};
GeluOutputs gelu_forward(const at::Tensor& x, bool keep) {
  const c10::hip::HIPGuard guard(x.get_device());
  check_channels(x);
  GeluOutputs g{at::empty(x.sizes(), plain(x)), keep ? packed_like(x) : Packed{}};
  const at::Tensor x2 = rows(x);
  const saf_tensor_t xd = rows_desc(kGelu, x2), yd = rows_desc(kGelu, g.y), qd = rows_desc(kGelu, g.p.q),
                     ed = rows_desc(kGelu, g.p.exp);
  check(lib.gelu(&xd, &yd, &qd, &ed, stream()));
  return g;
}
// (dx, gelu of the held values or undefined)
std::pair<at::Tensor, at::Tensor> gelu_backward(const at::Tensor& q, const at::Tensor& exp, const at::Tensor& dy, bool again) {
  const c10::hip::HIPGuard guard(dy.get_device());
  const at::Tensor g = rows(dy), dx = at::empty(q.sizes(), plain(dy)), y = again ? at::empty(q.sizes(), plain(dy)) : at::Tensor();
  const saf_tensor_t qd = rows_desc(kGelu, q), ed = rows_desc(kGelu, exp), gd = rows_desc(kGelu, g),
                     xd = rows_desc(kGelu, dx), yd = rows_desc(kGelu, y);
  check(lib.gelu_bwd(&qd, &ed, &gd, &xd, &yd, stream()));
  return {dx, y};
}

struct GeluPacked : public torch::autograd::Function<GeluPacked> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x) {
    const GeluOutputs g = gelu_forward(x, true);
    ctx->save_for_backward({g.p.q, g.p.exp});
    ctx->set_materialize_grads(false);
    return {g.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor()};
    const auto saved = ctx->get_saved_variables();
    at::Tensor dx;
    {
      at::NoGradGuard no_grad;
      dx = gelu_backward(saved[0], saved[1], grads[0], false).first;
    }
    return {only_once(kGelu, dx)};
  }
};

PyObject* wrap_all(std::initializer_list<at::Tensor> ts) {
  PyObject* t = PyTuple_New((Py_ssize_t)ts.size());
  if (t == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& x : ts) PyTuple_SET_ITEM(t, i++, wrap(x));
  return t;
}

bool counted(const char* usage, Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_SetString(PyExc_TypeError, usage);
  else if (lib.embed == nullptr) PyErr_SetString(PyExc_RuntimeError, "libsafattn.so is not loaded");
  return n == want && lib.embed != nullptr;
}

}  // namespace

PyObject* embed_tokens(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted("embed_tokens(tokens, weight, scale, ignore_index, dtype)", n, 5)) return nullptr;
  const at::Tensor &tokens = tensor(kEmbed, args[0]), &weight = tensor(kEmbed, args[1]);
  same_device(kEmbed, tokens, weight);
  TORCH_CHECK_VALUE(weight.dim() == 2, kEmbed, ": weight must be (V, C)");
  const EmbedOptions o{PyFloat_AsDouble(args[2]), PyLong_AsLongLong(args[3]),
                       type_of(PyLong_AsLong(args[4]), weight.scalar_type())};
  if (PyErr_Occurred()) return nullptr;
  if (!recorded(weight)) return wrap(embed_forward(tokens, weight, o));
  refuse_foreign_capture(kEmbed, "weights", weight);
  return wrap(EmbedTokens::apply(weight, tokens, o)[0]);
  END_HANDLE_TH_ERRORS
}

PyObject* add_layernorm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted("add_layernorm(x, delta, weight, bias, eps, dtype)", n, 6)) return nullptr;
  const at::Tensor &x = tensor(kNorm, args[0]), &weight = tensor(kNorm, args[2]);
  std::optional<at::Tensor> delta, bias;
  if (args[1] != Py_None) delta = tensor(kNorm, args[1]);
  if (args[3] != Py_None) bias = tensor(kNorm, args[3]);
  TORCH_CHECK_VALUE(x.dim() >= 1, kNorm, ": x must have channels");
  check_vector(kNorm, "weight", weight);
  if (bias) check_vector(kNorm, "bias", *bias);
  same_device(kNorm, weight, x);
  if (delta) {
    same_device(kNorm, *delta, x);
    TORCH_CHECK_VALUE(delta->sizes() == x.sizes(), kNorm, ": x and delta must share a shape (got ", x.sizes(), " and ",
                      delta->sizes(), ")");
  }
  if (bias) same_device(kNorm, *bias, x);
  const NormOptions o{PyFloat_AsDouble(args[4]),
                      type_of(PyLong_AsLong(args[5]), delta ? delta->scalar_type() : x.scalar_type())};
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor *leaves[4] = {&x, &weight, delta ? &*delta : nullptr, bias ? &*bias : nullptr};
  const char* names[4] = {"residuals", "weights", "additions", "biases"};
  bool grad = false;
  for (int i = 0; i < 4; ++i)
    if (leaves[i] != nullptr && recorded(*leaves[i])) {
      grad = true;
      refuse_foreign_capture(kNorm, names[i], *leaves[i]);
    }
  if (!grad) {
    const NormOutputs out = norm_forward(x, weight, delta ? *delta : at::Tensor(), bias ? *bias : at::Tensor(), o, false);
    return wrap_all({out.r, out.y});
  }
  const auto out = AddLayernorm::apply(x, weight, delta, bias, o);
  return delta ? wrap_all({out[0], out[1]}) : wrap_all({at::Tensor(), out[0]});
  END_HANDLE_TH_ERRORS
}

PyObject* gelu_packed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted("gelu_packed(x, keep)", n, 2)) return nullptr;
  const at::Tensor& x = tensor(kGelu, args[0]);
  same_device(kGelu, x, x);
  if (PyObject_IsTrue(args[1]) == 1) {
    at::NoGradGuard no_grad;
    const GeluOutputs g = gelu_forward(x, true);
    return wrap_all({g.y, g.p.q, g.p.exp});
  }
  if (!recorded(x)) return wrap(gelu_forward(x, false).y);
  refuse_foreign_capture(kGelu, "activations", x);
  return wrap(GeluPacked::apply(x)[0]);
  END_HANDLE_TH_ERRORS
}

PyObject* gelu_packed_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counted("gelu_packed_bwd(q, exp, dy, again)", n, 4)) return nullptr;
  const at::Tensor &q = tensor(kGelu, args[0]), &exp = tensor(kGelu, args[1]), &dy = tensor(kGelu, args[2]);
  same_device(kGelu, q, dy);
  same_device(kGelu, exp, dy);
  at::NoGradGuard no_grad;
  const auto [dx, y] = gelu_backward(q, exp, dy, PyObject_IsTrue(args[3]) == 1);
  return wrap_all({dx, y});
  END_HANDLE_TH_ERRORS
}

PyObject* pack_activation(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* what = "pack_activation";
  if (!counted("pack_activation(x)", n, 1)) return nullptr;
  const at::Tensor& x = tensor(what, args[0]);
  same_device(what, x, x);
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded(x), what, " has no backward: call it under torch.no_grad()");
  const c10::hip::HIPGuard guard(x.get_device());
  check_channels(x);
  const Packed p = packed_like(x);
  const at::Tensor x2 = rows(x);
  const saf_tensor_t xd = rows_desc(what, x2), qd = rows_desc(what, p.q), ed = rows_desc(what, p.exp);
  check(lib.pack(&xd, &qd, &ed, stream()));
  return wrap_all({p.q, p.exp});
  END_HANDLE_TH_ERRORS
}

PyObject* unpack_activation(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  constexpr const char* what = "unpack_activation";
  if (!counted("unpack_activation(q, exp, dtype)", n, 3)) return nullptr;
  const at::Tensor &q = tensor(what, args[0]), &exp = tensor(what, args[1]);
  const long code = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  same_device(what, q, q);
  same_device(what, exp, q);
  TORCH_CHECK_VALUE(q.dim() >= 1 && q.is_contiguous() && exp.is_contiguous(), what, ": q and exp must be contiguous");
  const c10::hip::HIPGuard guard(q.get_device());
  const at::Tensor y = at::empty(q.sizes(), plain(q).dtype(type_of(code, at::kFloat)));
  const saf_tensor_t qd = rows_desc(what, q), ed = rows_desc(what, exp), yd = rows_desc(what, y);
  check(lib.unpack(&qd, &ed, &yd, stream()));
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* check_differentiable(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = n > 0 ? PyUnicode_AsUTF8(args[0]) : nullptr;
  if (what == nullptr) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "check_differentiable(what, *tensors)");
    return nullptr;
  }
  for (Py_ssize_t i = 1; i < n; ++i) {
    if (args[i] == Py_None) continue;
    const at::Tensor& x = tensor(what, args[i]);
    same_device(what, x, THPVariable_Unpack(args[1]));
    if (recorded(x)) refuse_foreign_capture(what, "inputs", x);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* library_train(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 10) {
    PyErr_SetString(PyExc_TypeError, "library_train(10 addresses)");
    return nullptr;
  }
  void* p[10];
  for (int i = 0; i < 10; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  lib.embed = reinterpret_cast<decltype(lib.embed)>(p[0]);
  lib.embed_bwd = reinterpret_cast<decltype(lib.embed_bwd)>(p[1]);
  lib.embed_bytes = reinterpret_cast<decltype(lib.embed_bytes)>(p[2]);
  lib.layernorm = reinterpret_cast<decltype(lib.layernorm)>(p[3]);
  lib.layernorm_bwd = reinterpret_cast<decltype(lib.layernorm_bwd)>(p[4]);
  lib.layernorm_bytes = reinterpret_cast<decltype(lib.layernorm_bytes)>(p[5]);
  lib.pack = reinterpret_cast<decltype(lib.pack)>(p[6]);
  lib.unpack = reinterpret_cast<decltype(lib.unpack)>(p[7]);
  lib.gelu = reinterpret_cast<decltype(lib.gelu)>(p[8]);
  lib.gelu_bwd = reinterpret_cast<decltype(lib.gelu_bwd)>(p[9]);
  Py_RETURN_NONE;
}

}  // namespace saf_bind
