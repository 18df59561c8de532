// _srxhost: the host side of the calls whose Python would cost more than their kernels.
//
//   resnorm(...)   residual.py's operator: argument checks, memory order, outputs, the autograd node (its backward pass runs
//                  without Python), and the calls of libsrx's srx_resnorm_* entry points.
//   gather(...)    optim.py's lists: addresses and types of hundreds of parameters and gradients in one pass.
//   unheld(...)    finds a tensor whose storage does not hold it.
//   written(...)   tells autograd that a step has written those parameters.
//   bind(...)      the addresses of libsrx's entry points (the library that _lib.py has loaded).
//
// libsrx itself stays free of torch: this module is to it what the ctypes binding is, for tensors.
#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/custom_class.h>
#include "srx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

// ------------------------------------------------------------------------------------------------ errors
struct Refused {            // becomes a Python exception of that type
  PyObject* type;
  std::string msg;
};
template <typename... A> [[noreturn]] void refuse(PyObject* type, const A&... a) { throw Refused{type, c10::str(a...)}; }

template <typename F> PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.msg.c_str());
  } catch (...) {           // torch's own: a Python exception from a hook, out of memory, ... keep their types
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// ------------------------------------------------------------------------------------------------ what cannot follow these calls
// A trace records torch's own operations: it would hold the allocation of the outputs and nothing that writes them.
void need_untraced(const char* what) {
  const bool proxies = c10::impl::TorchDispatchModeTLS::any_modes_set() &&
                       c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
  if (torch::jit::tracer::isTracing() || proxies || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch))
    refuse(PyExc_RuntimeError, what, " cannot be traced (torch.jit.trace, make_fx, torch.export): its kernels are no torch operations");
}
// A tangent (torch.autograd.forward_ad) would be dropped.
void need_no_tangent(const variable_list& given) {
  for (const Tensor& t : given)
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
      refuse(PyExc_RuntimeError, "gated_residual and channel_norm have no forward-mode derivative: an input carries a tangent");
}

// ------------------------------------------------------------------------------------------------ libsrx
struct Lib {
  int (*resnorm_forward)(const srx_resnorm_desc*, void*);
  int (*resnorm_backward)(const srx_resnorm_desc*, void*);
  int64_t (*resnorm_ws_floats)(const srx_resnorm_desc*);
  const char* (*last_error)();
} lib;

void call(int (*fn)(const srx_resnorm_desc*, void*), const char* name, const srx_resnorm_desc& d, const c10::Device& dev) {
  const int rc = fn(&d, c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream());
  TORCH_CHECK(rc == 0, "libsrx ", name, " failed (status ", rc, "): ", lib.last_error());
}

// ------------------------------------------------------------------------------------------------ memory order
// How the channels and pixels of one call lie in memory; every tensor of the call is brought to it.
struct Order {
  bool rows;       // channels innermost
  bool moved;      // dim 1 is the channels and lies innermost
  int64_t B, C, P;
  std::vector<int64_t> shape;
};

Tensor channels_last(const Tensor& t) { return t.movedim(1, -1); }

// whether a tensor's storage holds all of it (a storage can be resized under its tensors; unstored zeros have one without memory)
bool held(const Tensor& t) {
  if (!t.numel()) return true;
  if (!t.storage().data()) return false;
  const size_t end = t.is_contiguous() ? (t.storage_offset() + t.numel()) * t.itemsize()
                                       : at::detail::computeStorageNbytes(t.sizes(), t.strides(), t.itemsize(), t.storage_offset());
  return end <= t.storage().nbytes();
}
void need_held(const Tensor& t) { TORCH_CHECK(held(t), "a tensor of shape ", t.sizes(), " whose memory has been freed"); }
// t with its values in memory: a view whose values are the negatives of what lies there, and a tensor of zeros without memory,
// are copied (both count as contiguous)
Tensor in_memory(const Tensor& t) {
  if (!t.defined() || t.layout() != at::kStrided) return t;
  if (t._is_zerotensor()) return t.clone();
  need_held(t);
  return t.is_neg() ? t.clone() : t;
}

Order order_of(const Tensor& x, int64_t channel_dim) {
  const int64_t dims = x.dim();
  if (!x.is_cuda()) refuse(PyExc_RuntimeError, "libsrx runs on a ROCm GPU only (input is on ", x.device(), ")");
  if (x.scalar_type() != at::kFloat && x.scalar_type() != at::kBFloat16)
    refuse(PyExc_TypeError, "float32 or bfloat16 tensors are supported, got ", x.scalar_type());
  if (dims < 2 || channel_dim < -dims || channel_dim >= dims)
    refuse(PyExc_ValueError, "channel_dim ", channel_dim, " of a tensor of shape ", x.sizes());
  const int64_t at = channel_dim < 0 ? channel_dim + dims : channel_dim;
  if (at != 1 && at != dims - 1) refuse(PyExc_ValueError, "channels must be at dim 1 or last, not at dim ", at, " of ", dims);
  Order o;
  o.shape = x.sizes().vec();
  o.B = x.size(0);
  o.C = x.size(at);
  if (o.C == 0) refuse(PyExc_ValueError, "no channels in a tensor of shape ", x.sizes());
  o.P = 1;
  for (int64_t i = 1; i < dims; ++i)
    if (i != at) o.P *= x.size(i);
  // channels at dim 1 that lie innermost in memory (channels-last maps), or a single pixel: rows
  o.moved = at != dims - 1 && (o.P == 1 || (!x.is_contiguous() && channels_last(x).is_contiguous()));
  o.rows = at == dims - 1 || o.moved;
  const int64_t most = o.rows ? SRX_RESNORM_MAX_ROWS_C : SRX_RESNORM_MAX_PLANES_C;
  if (o.C > most) refuse(PyExc_ValueError, o.C, " channels: at most ", most, " are supported ", o.rows ? "channels last" : "in maps");
  if (o.B >= (1LL << 31) || o.P >= (1LL << 31)) refuse(PyExc_ValueError, "sizes of 2^31 and more are not supported: ", x.sizes());
  return o;
}

// t in that order: t itself where its strides fit, else a copy; its row / image stride
Tensor taken(const Order& o, const Tensor& t, int64_t& stride) {
  if (o.rows) {
    Tensor v = o.moved ? channels_last(t) : t;
    stride = o.C;
    if (v.is_contiguous()) return v;
    bool fits = o.C == 1 || v.stride(-1) == 1;       // one stride between all rows?
    int64_t step = -1, next = 0;
    for (int64_t i = v.dim() - 2; i >= 0 && fits; --i) {
      if (v.size(i) == 1) continue;
      if (step < 0) step = v.stride(i);
      else fits = v.stride(i) == next;
      next = v.stride(i) * v.size(i);
    }
    if (!fits || step == 0) return v.contiguous();       // (a row that is expanded over others: copied)
    if (step > 0) stride = step;
    return v;
  }
  stride = o.C * o.P;
  if (t.is_contiguous()) return t;
  int64_t expect = stride;
  bool fits = true;
  for (int64_t i = 1; i < t.dim(); ++i) {
    expect /= std::max<int64_t>(t.size(i), 1);
    fits = fits && (t.size(i) == 1 || t.stride(i) == expect);
  }
  if (!fits) return t.contiguous();
  if (o.B > 1) stride = t.stride(0);
  return t;
}

Tensor fresh(const Order& o, const Tensor& like) {
  if (!o.moved) return at::empty(o.shape, like.options());
  std::vector<int64_t> s(o.shape);
  s.push_back(s[1]);
  s.erase(s.begin() + 1);
  return at::empty(s, like.options()).movedim(-1, 1);
}

// ------------------------------------------------------------------------------------------------ the operator
struct Call : torch::CustomClassHolder {
  srx_resnorm_desc d;       // kinds, sizes, layout, gate
  Order order;
  bool branch;
};

const void* address(const Tensor& t) {
  if (!t.numel()) return reinterpret_cast<const void*>(16);       // nothing is read from an empty tensor
  need_held(t);
  return t.data_ptr();
}

struct Put {                // tensors that have to live until the launch
  std::vector<Tensor> keep;
  const Order& order;
  template <typename P> void operator()(const Tensor& t, P& ptr, int64_t& stride) {
    if (!t.defined()) return;
    need_held(t);
    keep.push_back(taken(order, t, stride));
    ptr = const_cast<void*>(address(keep.back()));
  }
};
const float* vec(const Tensor& t) { return t.defined() ? static_cast<const float*>(address(t)) : nullptr; }

void put_common(Put& put, srx_resnorm_desc& d, const Tensor& gate, const Tensor& w_post, const Tensor& b_post, const Tensor& w_pre,
                const Tensor& b_pre) {
  if (d.gate_mode == 3) put(gate, d.gate, d.gate_stride);
  else if (gate.defined()) d.gate = address(gate);
  d.w_post = vec(w_post);
  d.b_post = vec(b_post);
  d.w_pre = vec(w_pre);
  d.b_pre = vec(b_pre);
}

variable_list forward(const Call& c, const Tensor& x, const Tensor& f, const Tensor& gate, const Tensor& w_post, const Tensor& b_post,
                      const Tensor& w_pre, const Tensor& b_pre) {
  srx_resnorm_desc d = c.d;
  Put put{{}, c.order};
  put(x, d.x, d.x_stride);
  put(f, d.f, d.f_stride);
  put_common(put, d, gate, w_post, b_post, w_pre, b_pre);
  const int64_t stride = c.order.rows ? c.order.C : c.order.C * c.order.P;
  variable_list out;
  if (c.branch) {
    out.push_back(fresh(c.order, x));
    d.y = const_cast<void*>(address(out.back()));
    d.y_stride = stride;
  }
  if (d.pre_kind) {
    out.push_back(fresh(c.order, x));
    d.h = const_cast<void*>(address(out.back()));
    d.h_stride = stride;
  }
  call(lib.resnorm_forward, "srx_resnorm_forward", d, x.device());
  return out;
}

Tensor plain(const Opt& t) { return t.has_value() ? *t : Tensor(); }

struct ResNorm : torch::autograd::Function<ResNorm> {
  static variable_list forward(AutogradContext* ctx, c10::intrusive_ptr<Call> c, const Opt& x, const Opt& f, const Opt& gate,
                               const Opt& w_post, const Opt& b_post, const Opt& w_pre, const Opt& b_pre) {
    const variable_list out = ::forward(*c, *x, plain(f), plain(gate), plain(w_post), plain(b_post), plain(w_pre), plain(b_pre));
    ctx->set_materialize_grads(false);
    // x is read again only to form y for h's gradient
    ctx->save_for_backward({c->d.pre_kind ? *x : Tensor(), plain(f), plain(gate), plain(w_post), plain(b_post), plain(w_pre), plain(b_pre)});
    ctx->saved_data["call"] = c10::IValue::make_capsule(c);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto holder = ctx->saved_data["call"].toCapsule();
    const Call& c = static_cast<const Call&>(*holder);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &f = saved[1], &gate = saved[2];
    const Tensor dy = in_memory(c.branch ? grads.front() : Tensor()), dh = in_memory(c.d.pre_kind ? grads.back() : Tensor());
    variable_list out(8);                       // of the call, x, f, gate, w_post, b_post, w_pre, b_pre
    if (!dy.defined() && !dh.defined()) return out;
    try {
      need_untraced("the backward pass of gated_residual and channel_norm");
      need_no_tangent(grads);
    } catch (const Refused& r) {
      TORCH_CHECK(false, r.msg);
    }
    // inputs that were given, in order, are the node's edges
    bool need[8] = {};
    size_t edge = 0;
    need[1] = ctx->needs_input_grad(edge++);
    for (int i = 1; i < 7; ++i)
      if (saved[i].defined()) need[i + 1] = ctx->needs_input_grad(edge++);
    const Tensor& like = f.defined() ? f : x;
    const c10::DeviceGuard guard(like.device());
    const bool second = at::GradMode::is_enabled();       // asked to differentiate this pass: its results refuse it
    {
      const at::AutoGradMode off(false);
      if (!dh.defined()) need[6] = need[7] = false;
      srx_resnorm_desc d = c.d;
      const int64_t stride = c.order.rows ? c.order.C : c.order.C * c.order.P;
      auto map = [&](int at, bool want, auto& ptr, int64_t& s) {
        if (!want) return;
        out[at] = fresh(c.order, like);
        ptr = const_cast<void*>(address(out[at]));
        s = stride;
      };
      map(1, need[1] && dh.defined(), d.dx, d.dx_stride);
      if (need[1] && !dh.defined()) out[1] = dy;          // without h, y's gradient is x's
      map(2, need[2], d.df, d.df_stride);
      map(3, need[3] && d.gate_mode == 3, d.dgate, d.dgate_stride);
      auto small = [&](int at, at::IntArrayRef shape) -> float* {
        if (!need[at]) return nullptr;
        out[at] = at::empty(shape, like.options().dtype(at::kFloat));
        return static_cast<float*>(const_cast<void*>(address(out[at])));
      };
      if (d.gate_mode == 1 || d.gate_mode == 2) d.dgate = small(3, gate.sizes());
      d.dw_post = small(4, {c.order.C});
      d.db_post = small(5, {c.order.C});
      d.dw_pre = small(6, {c.order.C});
      d.db_pre = small(7, {c.order.C});
      if (dh.defined() || need[2] || need[3] || need[4] || need[5]) {
        Put put{{}, c.order};
        if (dh.defined()) put(x, d.x, d.x_stride);
        else d.pre_kind = 0;
        put(f, d.f, d.f_stride);                          // y is formed again from x and f
        put_common(put, d, gate, saved[3], saved[4], saved[5], saved[6]);
        put(dy, d.dy, d.dy_stride);
        put(dh, d.dh, d.dh_stride);
        const int64_t floats = lib.resnorm_ws_floats(&d);
        TORCH_CHECK(floats >= 0, "libsrx srx_resnorm_ws_floats failed: ", lib.last_error());
        const Tensor ws = at::empty({std::max<int64_t>(floats, 1)}, like.options().dtype(at::kFloat));
        d.ws = ws.data_ptr<float>();
        call(lib.resnorm_backward, "srx_resnorm_backward", d, like.device());
      }
    }
    if (second) {
      variable_list real;
      for (const Tensor& t : out)
        if (t.defined()) real.push_back(t.detach().requires_grad_());
      const auto once = std::make_shared<torch::autograd::DelayedError>("gated_residual and channel_norm can be differentiated once only", (int64_t)real.size());
      real = (*once)(std::move(real));
      size_t k = 0;
      for (Tensor& t : out)
        if (t.defined()) t = real[k++];
    }
    return out;
  }
};

Tensor channel_vector(const Tensor& t, const Order& o, const Tensor& x, const char* what) {
  if (!t.defined()) return t;
  if (t.dim() != 1 || t.size(0) != o.C || t.device() != x.device() || !t.is_floating_point())
    refuse(PyExc_ValueError, what, ": ", o.C, " values on ", x.device(), " expected, got ", t.scalar_type(), " of shape ", t.sizes(), " on ", t.device());
  return in_memory(t).to(at::kFloat).contiguous();
}

// Autograd keeps one accumulator per leaf for as long as any graph of that leaf lives, whoever recorded it, bound to the stream
// that the first of them was recorded on.  A backward pass captured on another stream would then make the capture wait for that
// stream, and ROCm's runtime ends the process when such a capture closes.  So the forward call is refused instead.
void need_own_accumulators(const variable_list& inputs, const c10::Device& dev) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const c10::Stream stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).unwrap();
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    if (accumulator && accumulator->stream() != stream)
      refuse(PyExc_RuntimeError,
             "a graph that was recorded before this capture, on another stream, still holds one of these leaves (an output of an "
             "earlier call is alive): delete it, or capture on the stream that it was recorded on");
  }
}

Tensor tensor_arg(PyObject* o, const char* what) {
  if (o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, what, " must be a tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(PyExc_TypeError, "a number expected, got ", Py_TYPE(o)->tp_name);
  }
  return v;
}

// resnorm(x, f, gate, w_post, b_post, w_pre, b_pre, post_kind, pre_kind, post_eps, pre_eps, gate_act, scale, channel_dim)
PyObject* resnorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (n != 14) refuse(PyExc_TypeError, "resnorm takes 14 arguments");
    static const char* const names[] = {"x", "f", "gate", "post.weight", "post.bias", "pre.weight", "pre.bias"};
    variable_list given;             // before any copy or conversion: the graph's leaves
    for (int i = 0; i < 7; ++i) given.push_back(tensor_arg(a[i], names[i]));
    if (!given[0].defined()) refuse(PyExc_TypeError, "x must be a tensor");
    need_untraced("gated_residual and channel_norm");
    need_no_tangent(given);
    auto c = c10::make_intrusive<Call>();
    const Tensor x = in_memory(given[0]), f = in_memory(given[1]);
    Tensor gate = in_memory(given[2]);
    c->order = order_of(x, PyLong_AsLongLong(a[13]));
    const Order& o = c->order;
    c->branch = f.defined();
    auto same = [&](const Tensor& t, const char* what) {
      if (t.sizes() != x.sizes() || t.scalar_type() != x.scalar_type() || t.device() != x.device())
        refuse(PyExc_ValueError, what, ": ", x.scalar_type(), " of shape ", x.sizes(), " on ", x.device(), " expected, got ", t.scalar_type(), " of ",
               t.sizes(), " on ", t.device());
    };
    if (c->branch) same(f, "f");
    srx_resnorm_desc& d = c->d;
    d = {};
    d.dtype = x.scalar_type() == at::kBFloat16 ? SRX_BF16 : SRX_F32;
    d.layout = o.rows ? SRX_RESNORM_ROWS : SRX_RESNORM_PLANES;
    d.B = (int32_t)o.B;
    d.C = (int32_t)o.C;
    d.P = (int32_t)o.P;
    d.post_kind = (int32_t)PyLong_AsLong(a[7]);
    d.pre_kind = (int32_t)PyLong_AsLong(a[8]);
    d.post_eps = (float)float_arg(a[9]);
    d.pre_eps = (float)float_arg(a[10]);
    d.scale = (float)float_arg(a[12]);
    if (gate.defined()) {
      if (gate.sizes() == x.sizes() && (gate.scalar_type() == x.scalar_type() || x.dim() > 2)) {       // [B, C] with another type: one for each of B
        same(gate, "gate");
        d.gate_mode = 3;
      } else if ((gate.dim() == 1 && gate.size(0) == o.C) || (gate.dim() == 2 && gate.size(0) == o.B && gate.size(1) == o.C)) {
        if (gate.device() != x.device() || !gate.is_floating_point())
          refuse(PyExc_ValueError, "gate: floating-point values on ", x.device(), " expected, got ", gate.scalar_type(), " on ", gate.device());
        d.gate_mode = gate.dim() == 1 ? 1 : 2;
        gate = gate.to(at::kFloat).contiguous();
      } else {
        refuse(PyExc_ValueError, "gate of shape ", gate.sizes(), ": [", o.C, "], [", o.B, ", ", o.C, "] or ", x.sizes(), " expected");
      }
      d.gate_act = (int32_t)PyLong_AsLong(a[11]);
    }
    auto vector_arg = [&](int at) { return channel_vector(given[at], o, x, names[at]); };
    const Tensor w_post = vector_arg(3), b_post = vector_arg(4), w_pre = vector_arg(5), b_pre = vector_arg(6);
    if (PyErr_Occurred()) return nullptr;
    const variable_list inputs = {x, f, gate, w_post, b_post, w_pre, b_pre};
    bool grad = false;
    if (at::GradMode::is_enabled())
      for (const Tensor& t : inputs) grad = grad || (t.defined() && t.requires_grad());
    variable_list out;
    const c10::OptionalDeviceGuard guard(x.device());
    if (grad) {
      need_own_accumulators(given, x.device());
      auto opt = [](const Tensor& t) -> Opt { return t.defined() ? Opt(t) : std::nullopt; };
      out = ResNorm::apply(c, opt(x), opt(f), opt(gate), opt(w_post), opt(b_post), opt(w_pre), opt(b_pre));
    } else {
      out = forward(*c, x, f, gate, w_post, b_post, w_pre, b_pre);
    }
    if (out.size() == 1) return THPVariable_Wrap(out[0]);
    PyObject* pair = PyTuple_New(2);
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out[0]));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(out[1]));
    return pair;
  });
}

// ------------------------------------------------------------------------------------------------ optim.py's lists
enum { GATHER_MOVED = 1, GATHER_ODD = 2, GATHER_BF16 = 4 };

struct Buffer {
  Py_buffer b;
  explicit Buffer(PyObject* o, Py_ssize_t bytes, const char* what) {
    if (PyObject_GetBuffer(o, &b, PyBUF_WRITABLE) != 0) {
      PyErr_Clear();
      refuse(PyExc_TypeError, what, " must be a writable buffer");
    }
    if (b.len < bytes) {
      PyBuffer_Release(&b);
      refuse(PyExc_ValueError, what, " must hold ", bytes, " bytes");
    }
  }
  ~Buffer() { PyBuffer_Release(&b); }
  Buffer(const Buffer&) = delete;
};

// gather(params, grads or None, bound, addresses, types, device index) -> flags.  Compares the parameters with bound[2 n]
// (uint64: addresses, then elements times two, plus one for bf16), and writes the gradients' addresses (uint64[n], 0: none)
// and types (uint8[n]).  GATHER_MOVED: a parameter's address, size or type differs, or it is not contiguous or a negative view.
// GATHER_ODD: a gradient cannot be taken as it is (shape, type, device, order, a negative view, no memory) and the caller has to look.
// GATHER_BF16: some gradient is bf16.  grads None: each parameter's .grad.
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 6) refuse(PyExc_TypeError, "gather takes 6 arguments");
    if (!PyList_Check(a[0]) || (a[1] != Py_None && !PyList_Check(a[1]))) refuse(PyExc_TypeError, "lists expected");
    need_untraced("AdamW.step");
    const Py_ssize_t n = PyList_GET_SIZE(a[0]);
    const bool given = a[1] != Py_None;
    if (given && PyList_GET_SIZE(a[1]) != n) refuse(PyExc_ValueError, PyList_GET_SIZE(a[1]), " gradients for ", n, " parameters");
    const Buffer bound(a[2], n * 16, "bound"), addresses(a[3], n * 8, "addresses"), types(a[4], n, "types");
    const long index = PyLong_AsLong(a[5]);
    if (PyErr_Occurred()) return nullptr;
    const auto* was = static_cast<const uint64_t*>(bound.b.buf);
    auto* to = static_cast<uint64_t*>(addresses.b.buf);
    auto* ty = static_cast<uint8_t*>(types.b.buf);
    const Tensor none;
    long flags = 0;
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_Check(PyList_GET_ITEM(a[0], i))) refuse(PyExc_TypeError, "parameter ", i, " is not a tensor");
      const Tensor& p = THPVariable_Unpack(PyList_GET_ITEM(a[0], i));
      if (reinterpret_cast<uint64_t>(p.data_ptr()) != was[i] || 2 * (uint64_t)p.numel() + (p.scalar_type() == at::kBFloat16) != was[n + i] ||
          !p.is_contiguous() || p.is_neg())
        flags |= GATHER_MOVED;
      to[i] = 0;
      ty[i] = SRX_F32;
      PyObject* go = given ? PyList_GET_ITEM(a[1], i) : nullptr;
      if (given && go != Py_None && !THPVariable_Check(go)) refuse(PyExc_TypeError, "gradient ", i, " is a ", Py_TYPE(go)->tp_name, ", not a tensor");
      const Tensor& g = !given ? p.grad() : go == Py_None ? none : THPVariable_Unpack(go);
      if (!g.defined()) continue;
      if (g.layout() != at::kStrided || g.is_neg() || g.sizes() != p.sizes() || g.device().index() != index || g.device().type() != p.device().type() ||
          (g.scalar_type() != at::kFloat && g.scalar_type() != at::kBFloat16) || !g.is_contiguous() || !held(g)) {
        flags |= GATHER_ODD;
        continue;
      }
      to[i] = g.numel() ? reinterpret_cast<uint64_t>(g.data_ptr()) : 16;         // an empty tensor takes its step too
      if (g.scalar_type() == at::kBFloat16) {
        ty[i] = SRX_BF16;
        flags |= GATHER_BF16;
      }
    }
    return PyLong_FromLong(flags);
  });
}

// unheld(tensors) -> the first one whose storage does not hold it, or -1
PyObject* unheld(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 1 || !PyList_Check(a[0])) refuse(PyExc_TypeError, "a list expected");
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[0]); ++i) {
      if (!THPVariable_Check(PyList_GET_ITEM(a[0], i))) refuse(PyExc_TypeError, "element ", i, " is not a tensor");
      if (!held(THPVariable_Unpack(PyList_GET_ITEM(a[0], i)))) return PyLong_FromSsize_t(i);
    }
    return PyLong_FromLong(-1);
  });
}

// written(params, addresses or None, others): advances the version counters of the parameters with an address (None: of
// all) and, if there was one, of the other tensors, as an in-place operation would: a graph that saved one of them then refuses its
// backward pass.  (Tensors made in inference mode have no counter and cannot be saved.)
PyObject* written(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  return guarded([&]() -> PyObject* {
    if (nargs != 3) refuse(PyExc_TypeError, "written takes 3 arguments");
    if (!PyList_Check(a[0]) || !PyList_Check(a[2])) refuse(PyExc_TypeError, "lists expected");
    const Py_ssize_t n = PyList_GET_SIZE(a[0]);
    std::optional<Buffer> addresses;
    if (a[1] != Py_None) addresses.emplace(a[1], n * 8, "addresses");
    const auto* at = addresses ? static_cast<const uint64_t*>(addresses->b.buf) : nullptr;
    auto bump = [](PyObject* list, Py_ssize_t i) {
      if (!THPVariable_Check(PyList_GET_ITEM(list, i))) refuse(PyExc_TypeError, "element ", i, " is not a tensor");
      const Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(list, i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    bool any = false;
    for (Py_ssize_t i = 0; i < n; ++i)
      if (!at || at[i]) {
        bump(a[0], i);
        any = true;
      }
    for (Py_ssize_t i = 0; any && i < PyList_GET_SIZE(a[2]); ++i) bump(a[2], i);
    Py_RETURN_NONE;
  });
}

// bind(srx_resnorm_forward, srx_resnorm_backward, srx_resnorm_ws_floats, srx_last_error): their addresses
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "bind takes 4 addresses");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  lib.resnorm_forward = reinterpret_cast<decltype(lib.resnorm_forward)>(p[0]);
  lib.resnorm_backward = reinterpret_cast<decltype(lib.resnorm_backward)>(p[1]);
  lib.resnorm_ws_floats = reinterpret_cast<decltype(lib.resnorm_ws_floats)>(p[2]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(p[3]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"resnorm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(resnorm)), METH_FASTCALL, nullptr},
                         {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gather)), METH_FASTCALL, nullptr},
                         {"unheld", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(unheld)), METH_FASTCALL, nullptr},
                         {"written", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(written)), METH_FASTCALL, nullptr},
                         {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_srxhost", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__srxhost() {
  PyObject* m = PyModule_Create(&module);
  if (m) PyModule_AddIntConstant(m, "desc_bytes", (long)sizeof(srx_resnorm_desc));
  return m;
}
