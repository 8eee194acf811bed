// gdino_amd._host: the host side of the operators whose calls are shorter than
// Python takes to describe them (gdino_amd.linear, gdino_amd.optim).
//
// A feed-forward layer of a few tokens or an optimizer step over a small head
// runs a few microseconds on the device; checking and handing over its tensors
// from Python costs 10 to 25, a backward through a Python function some 60 more
// (the autograd thread waits for the interpreter), and an optimizer step has thousands of
// tensors to ask at 0.1 us a question.  Here the checks, the outputs and the
// call to the C-ABI (include/gdino_amd.h) take one to five.
//
// The library is not linked: bind() receives its entry points' addresses from
// gdino_amd._lib, which loads it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../../include/gdino_amd.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------ the library
struct Api {
  decltype(&gd_last_error) last_error;
  decltype(&gd_linear_readable) linear_readable;
  decltype(&gd_linear_pack) linear_pack;
  decltype(&gd_linear_forward_workspace_bytes) linear_forward_bytes;
  decltype(&gd_linear_forward) linear_forward;
  decltype(&gd_linear_backward_workspace_bytes) linear_backward_bytes;
  decltype(&gd_linear_backward) linear_backward;
  decltype(&gd_adamw_step) adamw_step;
  decltype(&gd_grad_norm_workspace_bytes) grad_norm_bytes;
  decltype(&gd_grad_norm) grad_norm;
};
Api api;

void run(const char* name, gd_status status) {
  TORCH_CHECK(status == GD_OK, name, ": status ", int(status), ": ", api.last_error());
}

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return GD_F32;
    case at::kBFloat16: return GD_BF16;
    case at::kHalf: return GD_F16;
    default: return -1;
  }
}

// the current stream of the tensor's device (host tensors, which only the kernels' emulator takes: none)
gd_stream_t stream_of(const Tensor& t) {
  return t.is_cuda() ? reinterpret_cast<gd_stream_t>(c10::hip::getCurrentHIPStream(t.get_device()).stream()) : nullptr;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({int64_t(bytes)}, like.options().dtype(at::kByte).requires_grad(false)) : Tensor();
}

const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* mut(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

constexpr const char* kWrapped = "it takes plain tensors, no wrappers around them (vmap, torch.func, FakeTensor, DTensor)";
bool wrapped(const Tensor& t) {
  using c10::DispatchKey;
  static const c10::DispatchKeySet keys({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                         DispatchKey::Batched, DispatchKey::Functionalize});
  return t.key_set().has_any(keys);
}

// Why a call with these tensors cannot be made here and now, or NULL.  The operators are calls, not operations that torch
// sees: what records operations (torch.jit.trace, make_fx, torch.export) would keep the outputs' allocation and none
// of their values, and a dual tensor's tangent would be lost.  A wrapper (FakeTensor, DTensor, what vmap and torch.func
// hand on) has no memory to be read.
const char* obstacle(std::initializer_list<const Tensor*> tensors) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  const bool modes = Modes::any_modes_set();
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
      (modes && Modes::get_mode(Key::PROXY)))
    return "it cannot be traced (its kernels are not torch operations)";
  if (modes && (Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL))) return kWrapped;  // (its outputs would be)
  const bool forward_mode = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (wrapped(*t)) return kWrapped;
    if (forward_mode && t->_fw_grad(0).defined()) return "it has no forward-mode derivatives";
  }
  return nullptr;
}
void require_no_obstacle(const char* what, std::initializer_list<const Tensor*> tensors = {}) {
  const char* const why = obstacle(tensors);
  TORCH_CHECK(!why, what, ": ", why);
}

// ------------------------------------------------------------------ linear layer
// t as [rows, features] with the features contiguous
Tensor rows_of(const Tensor& t) {
  Tensor r = (t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})).resolve_neg();
  const int64_t cols = r.size(1), pitch = r.stride(0);
  const bool dense = r.stride(1) == 1 || cols == 1;
  // (a single row's pitch may be anything, and contiguous() leaves it)
  if (dense && pitch < cols && r.size(0) == 1) return r.as_strided({1, cols}, {cols, 1});
  return dense && pitch >= cols ? r : r.contiguous();
}

struct Forward {
  Tensor y, z, x, w;  // x, w: as the kernels read them, K wide or padded to 8
};

// x [M, K], w [N, K], r [M, N]: rows; y of `lead`'s dimensions, its last one N
Forward linear_forward(const Tensor& x0, const Tensor& w0, const Tensor& b, int act, const Tensor& r, bool want_z,
                       at::IntArrayRef lead) {
  Tensor x = x0, w = w0;
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  TORCH_CHECK_VALUE(m <= (1 << 30) && k <= (1 << 22) && n <= (1 << 22), "linear_act: over 2^30 rows or 2^22 features");
  const auto like = x.options().requires_grad(false);
  Forward f;
  c10::SmallVector<int64_t, 6> shape(lead.begin(), lead.end());
  shape.back() = n;
  f.y = at::empty(shape, r.defined() ? like.dtype(r.scalar_type()) : like);
  f.x = x;
  f.w = w;
  if (m == 0) return f;
  if (want_z) f.z = at::empty({m, (n + 7) / 8 * 8}, like);
  const c10::DeviceGuard guard(x.device());
  const bool pack_x = !api.linear_readable(data(x), x.stride(0), k, 0), pack_w = !api.linear_readable(data(w), w.stride(0), k, 0);
  if (pack_x || pack_w) {
    // (the copies also serve the backward)
    const int64_t k8 = (k + 7) / 8 * 8;
    if (pack_x) f.x = at::empty({m, k8}, like);
    if (pack_w) f.w = at::empty({n, k8}, like);
    run("gd_linear_pack", api.linear_pack(data(x), x.stride(0), pack_x ? m : 0, data(w), w.stride(0), pack_w ? n : 0, k,
                                          mut(f.x), mut(f.w), stream_of(x)));
    x = f.x;
    w = f.w;
  }
  const size_t bytes = api.linear_forward_bytes(m, k, n);
  const Tensor ws = workspace(bytes, x);
  const int code = code_of(x.scalar_type());
  run("gd_linear_forward",
      api.linear_forward(code, data(x), x.stride(0), data(w), w.stride(0), data(b), act, data(r),
                         r.defined() ? code_of(r.scalar_type()) : code, r.defined() ? r.stride(0) : 0, m, k, n, mut(f.y),
                         code_of(f.y.scalar_type()), n, mut(f.z), f.z.defined() ? f.z.stride(0) : 0, 1, mut(ws), bytes,
                         stream_of(x)));
  return f;
}

// x, weight, bias: what the gradients go to, in their own types; xc, wc, bc: what the kernels read
struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const std::optional<Tensor>& bias, const std::optional<Tensor>& residual, const Tensor& xc,
                        const Tensor& wc, const std::optional<Tensor>& bc, int64_t act) {
    const Tensor r = residual ? rows_of(*residual) : Tensor();
    const bool wants = x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad());
    // of a ReLU without a residual, y itself tells where z <= 0
    const bool by_y = act == 1 && !residual;
    const Tensor x2 = rows_of(xc);
    const Forward f = linear_forward(x2, wc, bc ? *bc : Tensor(), int(act), r, wants && act != 0 && !by_y,
                                     x.sizes());
    // x for W's gradient, W for x's, z or y for the slope
    ctx->save_for_backward({weight.requires_grad() ? f.x : Tensor(), x.requires_grad() ? f.w : Tensor(),
                            !wants || act == 0 ? Tensor() : by_y ? f.y : f.z});
    ctx->saved_data["x"] = x.sizes().vec();
    ctx->saved_data["call"] =
        std::vector<int64_t>{act, x2.size(0), weight.size(0), int64_t(x.scalar_type()), int64_t(weight.scalar_type()),
                             int64_t(xc.scalar_type()), bias.has_value(), residual.has_value()};
    return f.y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(8);
    const Tensor dy = grads[0];
    if (!dy.defined()) return out;
    require_no_obstacle("linear_act's gradient", {&dy});
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear_act: gradients of its gradients are not implemented");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1];
    const auto call = ctx->saved_data["call"].toIntVector(), shape = ctx->saved_data["x"].toIntVector();
    const int act = int(call[0]);
    const int64_t m = call[1], n = call[2], k = shape.back();
    const auto xt = at::ScalarType(call[3]), wt = at::ScalarType(call[4]), type = at::ScalarType(call[5]);
    const bool has_b = call[6], has_r = call[7];
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    const bool want_b = has_b && ctx->needs_input_grad(2), want_r = has_r && ctx->needs_input_grad(2 + has_b);
    const auto like = dy.options().requires_grad(false);
    Tensor dx, dw, db;
    if (want_x) dx = at::empty({m, k}, like.dtype(xt));
    if (want_w) dw = at::empty({n, k}, like.dtype(wt));
    if (want_b) db = at::empty({n}, like.dtype(wt));
    if (m == 0) {
      if (want_w) dw.zero_();
      if (want_b) db.zero_();
    } else if (want_x || want_w || want_b) {
      const Tensor g = rows_of(dy);
      Tensor z = saved[2];
      if (z.defined()) z = z.dim() == 2 ? z : z.reshape({m, -1});
      const c10::DeviceGuard guard(g.device());
      const size_t bytes = api.linear_backward_bytes(m, k, n, want_x, want_w, want_b);
      const Tensor ws = workspace(bytes, g);
      const auto pitch = [](const Tensor& t) { return t.defined() ? t.stride(0) : 0; };
      run("gd_linear_backward",
          api.linear_backward(code_of(type), act, data(g), code_of(g.scalar_type()), g.stride(0), data(z),
                              pitch(z), data(x), pitch(x), data(w), pitch(w), m, k, n, mut(dx), code_of(xt), k, mut(dw),
                              mut(db), code_of(wt), 1, mut(ws), bytes, stream_of(g)));
    }
    if (want_x) out[0] = dx.view(shape);
    out[1] = dw;
    if (has_b) out[2] = db;
    if (want_r) out[3] = dy;
    return out;
  }
};

// x [..., K], weight [N, K], bias [N], residual [..., N]; xc, wc, bc: their casts, undefined where they are read as
// they are
Tensor linear_act(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, Tensor xc, Tensor wc,
                  Tensor bc, int act) {
  require_no_obstacle("linear_act", {&x, &weight, &bias, &residual});
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.size(1) == x.size(-1) && weight.numel() > 0,
                    "linear_act: x ", x.sizes(), " and weight ", weight.sizes(), " do not match");
  const int64_t n = weight.size(0);
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == n), "linear_act: bias ", bias.sizes(), " for ",
                    n, " features");
  if (residual.defined()) {
    auto want = x.sizes().vec();
    want.back() = n;
    TORCH_CHECK_VALUE(residual.sizes().equals(want), "linear_act: residual ", residual.sizes(), " for an output of ",
                      at::IntArrayRef(want));
  }
  for (const Tensor* t : {&weight, &bias, &residual})
    TORCH_CHECK(!t->defined() || t->device() == x.device(), "linear_act: tensors on different devices");
  if (!xc.defined()) xc = x;
  if (!wc.defined()) wc = weight;
  if (!bc.defined()) bc = bias;
  const auto type = xc.scalar_type();
  TORCH_CHECK_TYPE((type == at::kBFloat16 || type == at::kHalf) && wc.scalar_type() == type &&
                       (!bc.defined() || bc.scalar_type() == type),
                   "gdino_amd linear_act: x ", x.scalar_type(), ", weight ", weight.scalar_type(),
                   ": bf16 or fp16, alike with the bias (under autocast also fp32)");
  TORCH_CHECK_TYPE(!bias.defined() || bias.scalar_type() == weight.scalar_type(), "gdino_amd linear_act: weight ",
                   weight.scalar_type(), " and its bias differ in type");
  TORCH_CHECK_TYPE(!residual.defined() || residual.scalar_type() == type || residual.scalar_type() == at::kFloat,
                   "gdino_amd linear_act: residual ", residual.scalar_type(), " with a product in ", type);
  const bool needs = at::GradMode::is_enabled() &&
                     (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()) ||
                      (residual.defined() && residual.requires_grad()));
  if (needs) {
    const auto opt = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    {
      const at::AutoGradMode off(false);
      wc = rows_of(wc);
      if (bc.defined()) bc = bc.resolve_neg().contiguous();
    }
    return LinearFunction::apply(x, weight, opt(bias), opt(residual), xc.detach(), wc.detach(),
                                 bc.defined() ? std::optional<Tensor>(bc.detach()) : std::nullopt, int64_t(act));
  }
  const at::AutoGradMode off(false);
  return linear_forward(rows_of(xc), rows_of(wc), bc.defined() ? bc.resolve_neg().contiguous() : bc, act,
                        residual.defined() ? rows_of(residual) : residual, false, x.sizes())
      .y;
}

// -------------------------------------------------------------- lists of tensors
struct List {
  const char* name = "";
  bool written = false;
  std::vector<Tensor> held;
  std::vector<uint64_t> at;
  std::vector<int64_t> size;
};

// the one or two types a list may have
struct Types {
  at::ScalarType a, b;
  Types(at::ScalarType one) : a(one), b(one) {}
  Types(at::ScalarType one, at::ScalarType other) : a(one), b(other) {}
};

// `list`: a list or tuple of contiguous tensors of one of `types`, alike, on one device (device: of the call, set by its
// first list); written: see require_apart; sizes: the elements each has to have
List list_of(const char* what, const char* name, PyObject* list, Types types,
             std::optional<at::Device>* device, bool written, const std::vector<int64_t>* sizes) {
  const bool tuple = PyTuple_Check(list);
  TORCH_CHECK_TYPE(tuple || PyList_Check(list), what, ": ", name, ": a list of tensors");
  const Py_ssize_t n = tuple ? PyTuple_GET_SIZE(list) : PyList_GET_SIZE(list);
  TORCH_CHECK_VALUE(!sizes || size_t(n) == sizes->size(), what, ": ", n, " ", name, " for ", sizes ? sizes->size() : 0,
                    " tensors");
  List out;
  out.name = name;
  out.written = written;
  out.held.reserve(n);
  out.at.resize(n);
  out.size.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = tuple ? PyTuple_GET_ITEM(list, i) : PyList_GET_ITEM(list, i);
    TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": ", name, " ", i, " is not a tensor but ", Py_TYPE(o)->tp_name);
    const Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK_TYPE(!wrapped(t), what, ": ", name, " ", i, ": ", kWrapped);
    TORCH_CHECK_VALUE(!t.is_neg(), what, ": ", name, " ", i, " is a negated view; resolve_neg() first");
    TORCH_CHECK(t.layout() == at::kStrided && t.is_contiguous(), name, " tensors have to be contiguous (", what, ")");
    TORCH_CHECK_TYPE((t.scalar_type() == types.a || t.scalar_type() == types.b) && (i == 0 || t.scalar_type() == out.held[0].scalar_type()),
                     "gdino_amd ", what, ": unsupported or mixed dtypes of ", name);
    if (!device->has_value()) *device = t.device();
    TORCH_CHECK(t.device() == **device, what, ": ", name, " are not all on the device of the first tensor");
    out.size[i] = t.numel();
    TORCH_CHECK_VALUE(!sizes || (*sizes)[i] == out.size[i], what, ": ", name, " and the weights differ in their numbers of elements");
    // (a tensor that is written stops sharing a lazy clone's memory first)
    out.at[i] = out.size[i] ? reinterpret_cast<uint64_t>(written ? t.mutable_data_ptr() : t.const_data_ptr()) : 0;
    out.held.push_back(t);
  }
  return out;
}

// What is written overlaps nothing: no tensor of its own list, and none of another (what is only read may overlap what is).
void require_apart(const char* what, std::initializer_list<const List*> lists) {
  struct Span {
    uint64_t begin, end;
    const List* list;
  };
  c10::SmallVector<const List*, 8> in_order(lists.begin(), lists.end());
  // (lists that are cut from buffers one after the other need no sorting then)
  const auto first = [](const List* l) { return l->at.empty() ? 0 : l->at[0]; };
  std::sort(in_order.begin(), in_order.end(), [&](const List* a, const List* b) { return first(a) < first(b); });
  c10::SmallVector<Span, 64> all;
  for (const List* l : in_order)
    for (size_t i = 0; i < l->at.size(); ++i)
      if (l->size[i]) all.push_back({l->at[i], l->at[i] + uint64_t(l->size[i]) * l->held[i].element_size(), l});
  const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
  if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);
  const Span *any = nullptr, *written = nullptr;  // what reaches furthest so far
  for (const Span& s : all) {
    const Span* const other = s.list->written ? any : written;
    if (other && s.begin < other->end) {
      TORCH_CHECK_VALUE(other->list != s.list, what, ": ", s.list->name,
                        " overlap in memory (or a tensor is listed twice), and they are updated");
      TORCH_CHECK_VALUE(false, what, ": ", other->list->name, " and ", s.list->name,
                        " overlap in memory, and one of them is updated");
    }
    if (!any || s.end > any->end) any = &s;
    if (s.list->written && (!written || s.end > written->end)) written = &s;
  }
}

const float* scalar_of(const char* what, const char* name, const Tensor& t, const at::Device& device) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat && t.numel() == 1, "gdino_amd ", what, ": ", name,
                   " is a one-element fp32 tensor");
  TORCH_CHECK(t.device() == device, what, ": ", name, " is on ", t.device(), ", the tensors are elsewhere");
  return t.const_data_ptr<float>();
}

Tensor tensor_of(PyObject* o) {
  if (!o || o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), "not a tensor but ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const c10::ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
  } catch (const c10::TypeError& e) {
    PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ---------------------------------------------------------------------- Python
PyObject* py_bind(PyObject*, PyObject* addresses) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK_TYPE(PyDict_Check(addresses), "bind: a dict of addresses");
    const auto get = [&](const char* name, auto& into) {
      PyObject* v = PyDict_GetItemString(addresses, name);
      TORCH_CHECK_VALUE(v && PyLong_Check(v), "bind: no address of ", name);
      into = reinterpret_cast<std::decay_t<decltype(into)>>(PyLong_AsUnsignedLongLong(v));
    };
    Api a;
    get("gd_last_error", a.last_error);
    get("gd_linear_readable", a.linear_readable);
    get("gd_linear_pack", a.linear_pack);
    get("gd_linear_forward_workspace_bytes", a.linear_forward_bytes);
    get("gd_linear_forward", a.linear_forward);
    get("gd_linear_backward_workspace_bytes", a.linear_backward_bytes);
    get("gd_linear_backward", a.linear_backward);
    get("gd_adamw_step", a.adamw_step);
    get("gd_grad_norm_workspace_bytes", a.grad_norm_bytes);
    get("gd_grad_norm", a.grad_norm);
    api = a;
    Py_RETURN_NONE;
  });
}

PyObject* py_linear_act(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK_TYPE(n == 8, "linear_act: x, weight, bias, residual, three casts, activation");
    Tensor t[7];
    for (int i = 0; i < 7; ++i) t[i] = tensor_of(args[i]);
    TORCH_CHECK_TYPE(t[0].defined() && t[1].defined(), "linear_act: x and weight are tensors");
    return THPVariable_Wrap(linear_act(t[0], t[1], t[2], t[3], t[4], t[5], t[6], int(PyLong_AsLong(args[7]))));
  });
}

PyObject* py_grad_norm(PyObject*, PyObject* list) {
  return guarded([&]() -> PyObject* {
    require_no_obstacle("grad_norm");
    std::optional<at::Device> device;
    const List g = list_of("grad_norm", "gradients", list, {at::kFloat, at::kBFloat16}, &device, false, nullptr);
    TORCH_CHECK_VALUE(!g.held.empty(), "grad_norm: no tensors");
    const int count = int(g.held.size());
    const c10::DeviceGuard guard(*device);
    const size_t bytes = api.grad_norm_bytes(count, g.size.data());
    const Tensor ws = workspace(bytes, g.held[0]);
    const Tensor out = at::empty({}, g.held[0].options().dtype(at::kFloat).requires_grad(false));
    run("gd_grad_norm", api.grad_norm(count, g.size.data(), code_of(g.held[0].scalar_type()), g.at.data(), mut(ws), bytes,
                                      static_cast<float*>(mut(out)), stream_of(out)));
    return THPVariable_Wrap(out);
  });
}

PyObject* py_adamw_step(PyObject*, PyObject* args) {
  PyObject *p, *g, *m, *v, *ms, *vs, *copies, *steps, *lr_dev, *norm;
  double step, lr, b1, b2, eps, decay, max_norm;
  unsigned int seed;
  if (!PyArg_ParseTuple(args, "OOOOOOOOdOdddddOdI", &p, &g, &m, &v, &ms, &vs, &copies, &steps, &step, &lr_dev, &lr, &b1,
                        &b2, &eps, &decay, &norm, &max_norm, &seed))
    return nullptr;
  return guarded([&]() -> PyObject* {
    const char* what = "adamw_step";
    require_no_obstacle(what);
    std::optional<at::Device> device;
    const List lp = list_of(what, "weights", p, {at::kFloat}, &device, true, nullptr);
    const auto* size = &lp.size;
    const List lg = list_of(what, "gradients", g, {at::kFloat, at::kBFloat16}, &device, false, size);
    const bool eight = ms != Py_None;
    TORCH_CHECK_VALUE(eight == (vs != Py_None), what, ": moments in 8 bits have two lists of scales");
    const Types moments = eight ? Types(at::kByte, at::kFloat8_e4m3fn) : Types(at::kFloat);
    const List lm = list_of(what, "exp_avgs", m, moments, &device, true, size);
    const List lv = list_of(what, "exp_avg_sqs", v, moments, &device, true, size);
    List lms, lvs, lc, ls;
    if (eight) {
      std::vector<int64_t> blocks(size->size());
      for (size_t i = 0; i < blocks.size(); ++i) blocks[i] = ((*size)[i] + 31) / 32;
      lms = list_of(what, "exp_avg_scales", ms, {at::kByte, at::kFloat8_e8m0fnu}, &device, true, &blocks);
      lvs = list_of(what, "exp_avg_sq_scales", vs, {at::kByte, at::kFloat8_e8m0fnu}, &device, true, &blocks);
    }
    if (copies != Py_None) lc = list_of(what, "copies", copies, {at::kBFloat16}, &device, true, size);
    if (steps != Py_None) {
      const std::vector<int64_t> ones(size->size(), 1);
      ls = list_of(what, "steps", steps, {at::kFloat}, &device, false, &ones);
    }
    if (lp.held.empty()) Py_RETURN_NONE;
    // (a list given twice; the common mistake, named by its place)
    for (size_t i = 0; i < size->size(); ++i) {
      if ((*size)[i] == 0) continue;
      const uint64_t of[] = {lp.at[i], lg.at[i], lm.at[i], lv.at[i], eight ? lms.at[i] : 0, eight ? lvs.at[i] : 0,
                             copies != Py_None ? lc.at[i] : 0};
      for (int a = 0; a < 7; ++a)
        for (int b = 0; b < a; ++b)
          TORCH_CHECK_VALUE(of[a] == 0 || of[a] != of[b], what, ": two lists share tensor ", i);
    }
    require_apart(what, {&lp, &lg, &lm, &lv, &lms, &lvs, &lc});
    const Tensor lrt = tensor_of(lr_dev), nt = tensor_of(norm);
    const float* lrp = lrt.defined() ? scalar_of(what, "lr", lrt, *device) : nullptr;
    const float* np = nt.defined() ? scalar_of(what, "total_norm", nt, *device) : nullptr;
    const c10::DeviceGuard guard(*device);
    run("gd_adamw_step",
        api.adamw_step(int(lp.held.size()), size->data(), lp.at.data(), code_of(lg.held[0].scalar_type()), lg.at.data(),
                       eight ? 8 : 32, lm.at.data(), lv.at.data(), eight ? lms.at.data() : nullptr,
                       eight ? lvs.at.data() : nullptr, copies != Py_None ? lc.at.data() : nullptr,
                       steps != Py_None ? ls.at.data() : nullptr, step, lr, lrp, b1, b2, eps, decay, np, max_norm, seed,
                       stream_of(lp.held[0])));
    for (const List* list : std::initializer_list<const List*>{&lp, &lc})
      for (const Tensor& t : list->held)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // (inference tensors have none)
    Py_RETURN_NONE;
  });
}

PyObject* py_obstacle(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const char* why = obstacle({});
    for (Py_ssize_t i = 0; i < n && !why; ++i) {
      const Tensor t = tensor_of(args[i]);
      why = obstacle({&t});
    }
    if (why) return PyUnicode_FromString(why);
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, "the library's entry points: {name: address}"},
    {"obstacle", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_obstacle)), METH_FASTCALL,
     "obstacle(tensor or None, ...): why an operator cannot be called with these here and now, or None"},
    {"linear_act", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_linear_act)), METH_FASTCALL,
     "linear_act(x, weight, bias, residual, x's, weight's and bias's casts or None, activation)"},
    {"grad_norm", py_grad_norm, METH_O, "grad_norm(gradients)"},
    {"adamw_step", py_adamw_step, METH_VARARGS,
     "adamw_step(weights, gradients, exp_avgs, exp_avg_sqs, scales, scales, copies, steps, step, lr tensor, lr, beta1, "
     "beta2, eps, weight_decay, total_norm, max_norm, seed)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
