// The sequence operators on torch tensors, with their gradients as C++ autograd nodes (sequence.py and optim.py are its callers and hold the documentation).
//
// A call of these operators on one token or a short signal is a few microseconds of kernels.  Written in Python over ctypes, descriptor, checks and
// workspace took 14 to 20 us, an autograd function 50 to 80 more (its backward waits for the interpreter on another thread), and the tables of a norm over 367
// tensors 126 us.  So this layer is compiled; what it calls is the C ABI, whose addresses `bind` is given from the library that is already loaded.
#include <unordered_set>
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/graph_task.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include "../../include/vmm_kernels.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

#define VMM_BOUND(X) X(gated_scan_states) X(gated_scan_workspace) X(gated_scan) X(gated_scan_bwd) X(gated_ff_workspace) X(gated_ff) X(gated_ff_bwd) \
  X(grad_norm_workspace) X(grad_norm) X(grad_clip) X(adam_step_clipped)
struct Entries {
#define X(name) decltype(&vmm_##name) name = nullptr;
  VMM_BOUND(X)
#undef X
} lib;

// becomes videometamaterials_amd._native.NativeError
struct NativeFault : std::runtime_error { using std::runtime_error::runtime_error; };
// becomes NotImplementedError
struct Unsupported : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename E, typename... Args>
[[noreturn]] void fail(const Args&... args) { throw E(c10::str(args...)); }

void check(int code, const char* what) {
  if (code != 0) fail<NativeFault>(what, " failed with code ", code, " (hipError_t if > 0, rejected argument if < 0)");
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

void need_gpu(const Tensor& t, const char* what) {
  if (!t.is_cuda()) fail<NativeFault>(what, ": tensors must live on the GPU (there is no CPU path)");
}

// What is computed through raw pointers has no derivative in forward mode (a tangent would vanish without a word), and no tensor can stand in for another
// (subclasses, the wrappers of torch.func, lazily negated views).
void need_plain(const Tensor& t, const char* what) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet stand_ins{DispatchKey::Python,      DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper, DispatchKey::Functionalize,
                                          DispatchKey::ZeroTensor, DispatchKey::Negative};
  if (t.unsafeGetTensorImpl()->_fw_grad(0, t).defined()) fail<Unsupported>(what, ": no forward-mode derivative");
  if (t.unsafeGetTensorImpl()->key_set().has_any(stand_ins)) fail<Unsupported>(what, ": plain tensors only (no subclass, torch.func transform or lazy negation)");
}
void need_plain(const Maybe& t, const char* what) {
  if (t) need_plain(*t, what);
}

// Nothing that records operations instead of running them sees these: a trace would hold empty buffers that nobody fills.
void need_eager(const char* what) {
  using c10::impl::TorchDispatchModeTLS;
  using c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) ||
      TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FUNCTIONAL) || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch))
    fail<Unsupported>(what, ": cannot be traced (torch.jit.trace, make_fx, torch.export, fake tensors)");
}

vmm_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

std::string shape(const Tensor& t) { return c10::str(t.sizes()); }

// `t` with neighbouring values in its last dimension and rows less than 2^22 values apart, as the kernels' 32-bit offsets need them (else a copy).  The stride of
// a dimension of one says nothing and may be anything, in a contiguous tensor too: it is neither looked at nor handed on.
Tensor rows_of(const Tensor& t) {
  return (t.stride(-1) == 1 || t.size(-1) <= 1) && (t.stride(-2) < (1 << 22) || t.size(-2) <= 1) ? t : t.contiguous();
}
// a gradient as its values are in memory (part of a conjugated complex one can come negated, to be)
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
int64_t row_stride(const Tensor& t) { return t.size(-2) > 1 ? t.stride(-2) : t.size(-1); }

template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
template <typename T>
T* ptr(const Maybe& t) { return t ? ptr<T>(*t) : nullptr; }

Tensor fp32(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
Tensor same(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }

template <typename D>
Tensor workspace(int64_t (*query)(const D*, int32_t), D& d, bool backward, const Tensor& like, const char* what) {
  const int64_t size = query(&d, backward);
  if (size < 0) fail<py::value_error>(what, ": a size is out of range");
  if (size == 0) return {};
  Tensor w = at::empty({size}, like.options().dtype(at::kByte));
  d.workspace = w.data_ptr();
  d.workspace_bytes = size;
  return w;
}

// gradients that may be handed on, but not differentiated a second time
variable_list once(variable_list grads, const char* what) {
  if (!c10::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const auto n = static_cast<int64_t>(grads.size());
  return torch::autograd::DelayedError(c10::str(what, ": trying to differentiate twice a function that is differentiable once"), n).apply(std::move(grads));
}

// A leaf hands its gradient over on the stream that its first graph was made on.  Where an eager graph of that leaf is still alive, made on the default stream, a captured
// backward would have to wait across to that stream, which no capture allows: it would end in the middle, and the process with it.
void need_capturable(const char* what) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto* const wanted = torch::autograd::get_current_graph_task_exec_info();  // (empty: everything is)
  std::vector<torch::autograd::Node*> next;
  std::unordered_set<torch::autograd::Node*> seen;
  const auto follow = [&](torch::autograd::Node& node) {
    for (const auto& edge : node.next_edges()) {
      if (!edge.function || !seen.insert(edge.function.get()).second) continue;
      if (wanted && !wanted->empty())
        if (const auto it = wanted->find(edge.function.get()); it == wanted->end() || !it->second.should_execute()) continue;
      next.push_back(edge.function.get());
    }
  };
  if (const auto node = torch::autograd::get_current_node()) follow(*node);
  while (!next.empty()) {
    torch::autograd::Node& node = *next.back();
    next.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(&node))
      if (const auto stream = node.stream(); stream && stream->id() == 0)
        fail<NativeFault>(what, ": a captured backward needs leaves that no eager graph on the default stream holds: release that graph first");
    follow(node);
  }
}

// ---- gated linear recurrence

const char* const SCAN = "gated_linear_scan";

template <typename P>
void place(const Tensor& t, P& p, int64_t& batch, int64_t& row) {
  if (!t.defined()) return;
  p = t.data_ptr();
  batch = t.size(0) > 1 ? t.stride(0) : 0;
  row = row_stride(t);
}

vmm_gated_scan_desc scan_desc(const Tensor& x, const Tensor& gate, const Maybe& lengths) {
  vmm_gated_scan_desc d = {};
  place(x, d.x, d.x_batch, d.x_row);
  place(gate, d.gate, d.gate_batch, d.gate_row);
  d.lengths = ptr<int32_t>(lengths);
  d.L = x.size(1);
  d.B = static_cast<int32_t>(x.size(0));
  d.D = static_cast<int32_t>(x.size(2));
  d.type = type_of(x);
  return d;
}

std::tuple<Tensor, Tensor, Tensor> scan_forward(const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& lengths, bool keep) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = same(x.sizes(), x), last = fp32({x.size(0), x.size(2)}, x), states;
  vmm_gated_scan_desc d = scan_desc(x, gate, lengths);
  place(y, d.y, d.y_batch, d.y_row);
  d.h0 = ptr<float>(h0);
  d.h_last = ptr<float>(last);
  if (keep) {
    states = fp32({std::max<int64_t>(lib.gated_scan_states(&d), 0)}, x);
    d.states = ptr<float>(states);
  }
  const Tensor work = workspace(lib.gated_scan_workspace, d, false, x, SCAN);
  check(lib.gated_scan(&d, stream_of(x)), "vmm_gated_scan");
  return {y, last, states};
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& h0, const Maybe& lengths) {
    ctx->set_materialize_grads(false);
    auto [y, last, states] = scan_forward(x, gate, h0, lengths, true);
    ctx->save_for_backward({x, gate, lengths ? *lengths : Tensor(), states});
    ctx->saved_data["state"] = h0.has_value();
    return {y, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate = saved[1], &lengths = saved[2], &states = saved[3];
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    Tensor dx, dgate, dh0;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      need_capturable(SCAN);
      const Tensor dy = grads[0].defined() ? rows_of(plain(grads[0])) : Tensor(), dlast = grads[1].defined() ? plain(grads[1]).contiguous() : Tensor();
      if (ctx->needs_input_grad(0)) dx = same(x.sizes(), x);
      if (ctx->needs_input_grad(1)) dgate = same(x.sizes(), x);
      if (ctx->saved_data["state"].toBool() && ctx->needs_input_grad(2)) dh0 = fp32({x.size(0), x.size(2)}, x);
      vmm_gated_scan_desc d = scan_desc(x, gate, lengths.defined() ? Maybe(lengths) : Maybe());
      place(dy, d.dy, d.dy_batch, d.dy_row);
      place(dx, d.dx, d.dx_batch, d.dx_row);
      place(dgate, d.dgate, d.dgate_batch, d.dgate_row);
      d.states = ptr<float>(states);
      d.dh_last = ptr<float>(dlast);
      d.dh0 = ptr<float>(dh0);
      const Tensor work = workspace(lib.gated_scan_workspace, d, true, x, SCAN);
      check(lib.gated_scan_bwd(&d, stream_of(x)), "vmm_gated_scan_bwd");
    }
    return once({dx, dgate, dh0, Tensor()}, SCAN);
  }
};

std::tuple<Tensor, Tensor> gated_linear_scan(Tensor x, Tensor gate, Maybe h0, Maybe lengths) {
  need_eager(SCAN);
  need_plain(x, SCAN);
  need_plain(gate, SCAN);
  need_plain(h0, SCAN);
  if (x.dim() != 3 || gate.sizes() != x.sizes()) fail<py::value_error>(SCAN, ": x and gate must be (B, L, D) and alike, got ", shape(x), " and ", shape(gate));
  if (type_of(x) < 0 || gate.scalar_type() != x.scalar_type())
    fail<py::type_error>(SCAN, ": x and gate must be float32, bfloat16 or float16 alike, got ", x.scalar_type(), " and ", gate.scalar_type());
  need_gpu(x, SCAN);
  const int64_t B = x.size(0), L = x.size(1), D = x.size(2);
  if (h0 && (h0->sizes() != at::IntArrayRef({B, D}) || !h0->is_floating_point()))
    fail<py::value_error>(SCAN, ": h0 must be a floating (", B, ", ", D, "), got ", h0->scalar_type(), " ", shape(*h0));
  if (lengths && (lengths->sizes() != at::IntArrayRef({B}) || !at::isIntegralType(lengths->scalar_type(), false)))
    fail<py::value_error>(SCAN, ": lengths must be (", B, ",) integers, got ", lengths->scalar_type(), " ", shape(*lengths));
  if (gate.device() != x.device() || (h0 && h0->device() != x.device()) || (lengths && lengths->device() != x.device()))
    fail<py::value_error>(SCAN, ": all tensors must be on ", x.device().str());
  if (std::max({B, D}) >= (1LL << 31)) fail<py::value_error>(SCAN, ": a size is out of range");
  if (h0) h0 = h0->to(at::kFloat).contiguous();
  if (lengths && lengths->scalar_type() != at::kInt) {  // (in 64 bits before L is compared with: it need not fit a narrow type; and from 2^63 on they are beyond any L)
    const Tensor wide = lengths->to(at::kLong);
    lengths = (lengths->scalar_type() == at::kUInt64 ? at::where(wide.lt(0), L, wide) : wide).clamp(0, L).to(at::kInt);
  }
  if (lengths) lengths = lengths->contiguous();
  x = rows_of(x);
  gate = rows_of(gate);
  if (c10::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (h0 && h0->requires_grad()))) {
    auto out = GatedScan::apply(x, gate, h0, lengths);
    return {out[0], out[1]};
  }
  auto [y, last, states] = scan_forward(x, gate, h0, lengths, false);
  return {y, last};
}

// ---- gated feed-forward product

const char* const FF = "gated_feed_forward";

vmm_gated_ff_desc ff_desc(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
  vmm_gated_ff_desc d = {};
  d.x = x.data_ptr();
  d.ldx = row_stride(x);
  d.w_gate = wg.data_ptr();
  d.w_up = wu.data_ptr();
  d.M = x.size(0);
  d.K = static_cast<int32_t>(x.size(1));
  d.F = static_cast<int32_t>(wg.size(0));
  d.type = type_of(x);
  d.act = static_cast<int32_t>(act);
  return d;
}

// what the backward needs of the products stays in fp32: rounded to 16 bits they would put an error of their own into every gradient
std::tuple<Tensor, Tensor> ff_forward(const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& bg, const Maybe& bu, int64_t act, bool keep) {
  const c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), F = wg.size(0);
  Tensor h = same({M, F}, x), pre;
  vmm_gated_ff_desc d = ff_desc(x, wg, wu, act);
  d.b_gate = ptr<void>(bg);
  d.b_up = ptr<void>(bu);
  d.h = h.data_ptr();
  d.ldh = F;
  if (keep) {
    pre = fp32({2, M, F}, x);
    d.g_pre = ptr<float>(pre);
    d.u_pre = d.g_pre + M * F;
  }
  const Tensor work = workspace(lib.gated_ff_workspace, d, false, x, FF);
  check(lib.gated_ff(&d, stream_of(x)), "vmm_gated_ff");
  return {h, pre};
}

struct GatedFF : torch::autograd::Function<GatedFF> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Maybe& bg, const Maybe& bu, int64_t act) {
    auto [h, pre] = ff_forward(x, wg, wu, bg, bu, act, true);
    ctx->save_for_backward({x, wg, wu, pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bg.has_value();
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &pre = saved[3];
    const bool bias = ctx->saved_data["bias"].toBool(), need_wg = ctx->needs_input_grad(1), need_wu = ctx->needs_input_grad(2);
    const bool need_bg = bias && ctx->needs_input_grad(3), need_bu = bias && ctx->needs_input_grad(4);
    Tensor dx, dwg, dwu, dbg, dbu;
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(x.device());
      need_capturable(FF);
      const Tensor dh = rows_of(plain(grads[0]));
      if (ctx->needs_input_grad(0)) dx = same(x.sizes(), x);
      if (need_wg || need_wu) dwg = same(wg.sizes(), x), dwu = same(wg.sizes(), x);
      if (need_bg) dbg = same({wg.size(0)}, x);
      if (need_bu) dbu = same({wg.size(0)}, x);
      vmm_gated_ff_desc d = ff_desc(x, wg, wu, ctx->saved_data["act"].toInt());
      d.g_pre = ptr<float>(pre);
      d.u_pre = d.g_pre + x.size(0) * wg.size(0);
      d.dh = dh.data_ptr();
      d.lddh = row_stride(dh);
      d.dx = ptr<void>(dx);
      d.lddx = dx.defined() ? row_stride(dx) : 0;
      d.dw_gate = ptr<void>(dwg);
      d.dw_up = ptr<void>(dwu);
      d.db_gate = ptr<void>(dbg);
      d.db_up = ptr<void>(dbu);
      const Tensor work = workspace(lib.gated_ff_workspace, d, true, x, FF);
      check(lib.gated_ff_bwd(&d, stream_of(x)), "vmm_gated_ff_bwd");
    }
    return once({dx, need_wg ? dwg : Tensor(), need_wu ? dwu : Tensor(), dbg, dbu, Tensor()}, FF);
  }
};

Tensor gated_feed_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Maybe& b_gate, const Maybe& b_up, int64_t act) {
  need_eager(FF);
  if (x.dim() < 1 || w_gate.dim() != 2 || w_up.sizes() != w_gate.sizes() || x.size(-1) != w_gate.size(1) || w_gate.numel() == 0)
    fail<py::value_error>(FF, ": x (..., K) and weights (F, K) do not fit: ", shape(x), ", ", shape(w_gate), ", ", shape(w_up));
  if (b_gate.has_value() != b_up.has_value()) fail<py::value_error>(FF, ": both biases or none");
  const int64_t F = w_gate.size(0), K = w_gate.size(1);
  const Tensor* every[5] = {&x, &w_gate, &w_up, b_gate ? &*b_gate : nullptr, b_up ? &*b_up : nullptr};
  const int n = b_gate ? 5 : 3;
  bool grad = false;
  for (int i = 0; i < n; ++i) need_plain(*every[i], FF);
  for (int i = 3; i < n; ++i)
    if (every[i]->sizes() != at::IntArrayRef({F})) fail<py::value_error>(FF, ": biases must be (", F, ",), got ", shape(*every[i]));
  for (int i = 0; i < n; ++i) {
    if (type_of(x) < 0 || every[i]->scalar_type() != x.scalar_type())
      fail<py::type_error>(FF, ": float32, bfloat16 or float16 tensors of one type, got ", x.scalar_type(), " and ", every[i]->scalar_type());
    grad |= every[i]->requires_grad();
  }
  need_gpu(x, FF);
  for (int i = 1; i < n; ++i)
    if (every[i]->device() != x.device()) fail<py::value_error>(FF, ": all tensors must be on ", x.device().str());
  if (std::max({K, F}) >= (1LL << 31)) fail<py::value_error>(FF, ": a size is out of range");
  const Tensor rows = rows_of(x.dim() == 2 ? x : x.reshape({-1, K}));
  const Tensor wg = w_gate.contiguous(), wu = w_up.contiguous();
  const Maybe bg = b_gate ? Maybe(b_gate->contiguous()) : b_gate, bu = b_up ? Maybe(b_up->contiguous()) : b_up;
  const Tensor h = c10::GradMode::is_enabled() && grad ? GatedFF::apply(rows, wg, wu, bg, bu, act) : std::get<0>(ff_forward(rows, wg, wu, bg, bu, act, false));
  if (x.dim() == 2) return h;
  at::DimVector sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = F;
  return h.view(sizes);
}

// ---- norm, clipping, optimizer

struct Listed {
  std::vector<const Tensor*> tensors;  // (borrowed from `own`)
  py::object own;                      // the sequence, alive as long as they are
};

const Tensor& tensor_of(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) fail<py::type_error>(what, ": expected tensors, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

Listed listed(const py::object& sequence, const char* what) {
  Listed l;
  l.own = py::reinterpret_steal<py::object>(PySequence_Fast(sequence.ptr(), "expected a sequence of tensors"));
  if (!l.own) throw py::error_already_set();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(l.own.ptr());
  l.tensors.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) l.tensors.push_back(&tensor_of(PySequence_Fast_GET_ITEM(l.own.ptr(), i), what));
  return l;
}

void check_grads(const std::vector<const Tensor*>& grads, const char* what) {
  need_eager(what);
  for (const Tensor* g : grads) need_plain(*g, what);
  for (const Tensor* g : grads)
    if (type_of(*g) < 0) fail<py::type_error>(what, ": float32, bfloat16 or float16 tensors, got ", g->scalar_type());
  for (const Tensor* g : grads)
    if (g->layout() != at::kStrided || !g->is_contiguous()) fail<py::value_error>(what, ": tensors must be contiguous");
  for (const Tensor* g : grads)
    if (g->device() != grads[0]->device()) fail<py::value_error>(what, ": the tensors are on several devices");
  need_gpu(*grads[0], what);
}

std::vector<vmm_grad_job> grad_jobs(const std::vector<const Tensor*>& grads) {
  std::vector<vmm_grad_job> jobs(grads.size());
  for (size_t i = 0; i < grads.size(); ++i) jobs[i] = {grads[i]->data_ptr(), grads[i]->numel(), type_of(*grads[i]), 0};
  return jobs;
}

// (norm, factor) on the device; max_norm <= 0: the factor is one
Tensor norm_and_factor(const std::vector<vmm_grad_job>& jobs, double max_norm, const Tensor& like) {
  const auto n = static_cast<int32_t>(jobs.size());
  const int64_t size = lib.grad_norm_workspace(jobs.data(), n);
  if (size < 0) fail<py::value_error>("gradient norm: a tensor that is not aligned to its type");
  Tensor work = at::empty({size / 8}, like.options().dtype(at::kDouble)), out = fp32({2}, like);
  check(lib.grad_norm(jobs.data(), n, 1.0f, static_cast<float>(max_norm), nullptr, work.data_ptr(), ptr<float>(out), stream_of(like)), "vmm_grad_norm");
  return out;
}

// written through raw pointers: whoever has saved the tensor finds out
void written(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

Tensor grad_norm(const py::object& grads) {
  const at::NoGradGuard no_grad;
  const Listed l = listed(grads, "grad_norm");
  if (l.tensors.empty()) return at::zeros({}, at::kFloat);
  check_grads(l.tensors, "grad_norm");
  const c10::DeviceGuard guard(l.tensors[0]->device());
  return norm_and_factor(grad_jobs(l.tensors), 0.0, *l.tensors[0]).select(0, 0);
}

Tensor clip_grad_norm(const py::object& grads, double max_norm) {
  const char* const what = "clip_grad_norm_";
  const at::NoGradGuard no_grad;
  const Listed l = listed(grads, what);
  if (l.tensors.empty()) return at::zeros({}, at::kFloat);
  check_grads(l.tensors, what);
  const c10::DeviceGuard guard(l.tensors[0]->device());
  const auto jobs = grad_jobs(l.tensors);
  const Tensor out = norm_and_factor(jobs, max_norm, *l.tensors[0]);
  const int code = lib.grad_clip(jobs.data(), static_cast<int32_t>(jobs.size()), ptr<float>(out), stream_of(out));
  if (code == -2) fail<py::value_error>(what, ": tensors overlap in memory");
  check(code, "vmm_grad_clip");
  for (const Tensor* g : l.tensors) written(*g);
  return out.select(0, 0);
}

// One update; grads None: every parameter's own.  Parameters without a gradient stay as they are; none at all has one: None.
Maybe clipped_adam(const py::object& params, const py::object& exp_avgs, const py::object& exp_avg_sqs, const py::object& grads, double lr, double beta1, double beta2,
                   double eps, double max_norm, int64_t step) {
  const char* const what = "ClippedAdam.step";
  const at::NoGradGuard no_grad;
  const Listed p = listed(params, what), m = listed(exp_avgs, what), v = listed(exp_avg_sqs, what);
  const size_t n = p.tensors.size();
  py::object held;
  if (!grads.is_none()) {
    held = py::reinterpret_steal<py::object>(PySequence_Fast(grads.ptr(), "expected a sequence of tensors"));
    if (!held) throw py::error_already_set();
    const auto given = static_cast<size_t>(PySequence_Fast_GET_SIZE(held.ptr()));
    if (given != n) fail<py::value_error>(what, ": ", given, " gradients for ", n, " parameters");
  }
  std::vector<size_t> at_;
  std::vector<const Tensor*> g;
  at_.reserve(n);
  g.reserve(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor* one = nullptr;
    if (grads.is_none()) {
      const Tensor& own = p.tensors[i]->grad();
      if (own.defined()) one = &own;
    } else if (PyObject* o = PySequence_Fast_GET_ITEM(held.ptr(), i); o != Py_None) {
      one = &tensor_of(o, what);
    }
    if (!one) continue;
    if (one->numel() != p.tensors[i]->numel()) fail<py::value_error>(what, ": gradients do not fit the parameters");
    at_.push_back(i);
    g.push_back(one);
  }
  if (g.empty()) return std::nullopt;
  check_grads(g, what);
  std::vector<vmm_clip_adam_job> jobs(g.size());
  for (size_t k = 0; k < g.size(); ++k) {
    const Tensor* own[3] = {p.tensors[at_[k]], m.tensors[at_[k]], v.tensors[at_[k]]};
    for (const Tensor* t : own) {
      need_plain(*t, what);
      if (t->device() != g[0]->device() || t->scalar_type() != at::kFloat || !t->is_contiguous() || t->numel() != g[k]->numel())
        fail<py::value_error>(what, ": parameters and moments must be contiguous float32 tensors of one size, on the gradients' device");
    }
    jobs[k] = {ptr<float>(*own[0]), g[k]->data_ptr(), ptr<float>(*own[1]), ptr<float>(*own[2]), g[k]->numel(), type_of(*g[k]), 0};
  }
  const c10::DeviceGuard guard(g[0]->device());
  const Tensor out = norm_and_factor(grad_jobs(g), max_norm, *g[0]);
  const int code = lib.adam_step_clipped(jobs.data(), static_cast<int32_t>(jobs.size()), lr, beta1, beta2, eps, step, 1.0f, ptr<float>(out), nullptr, stream_of(out));
  if (code == -2) fail<py::value_error>(what, ": parameters, moments or gradients overlap in memory");
  check(code, "vmm_adam_step_clipped");
  for (const size_t i : at_)
    for (const Tensor* t : {p.tensors[i], m.tensors[i], v.tensors[i]}) written(*t);
  return out.select(0, 0);
}

void bind(const py::dict& addresses) {
#define X(name) lib.name = reinterpret_cast<decltype(lib.name)>(addresses["vmm_" #name].cast<uintptr_t>());
  VMM_BOUND(X)
#undef X
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeFault& e) {
      py::set_error(py::module_::import("videometamaterials_amd._native").attr("NativeError"), e.what());
    } catch (const Unsupported& e) {
      py::set_error(PyExc_NotImplementedError, e.what());
    }
  });
  m.attr("entries") = [] {
    py::list names;
#define X(name) names.append("vmm_" #name);
    VMM_BOUND(X)
#undef X
    return names;
  }();
  m.def("bind", &bind);
  m.def("gated_linear_scan", &gated_linear_scan);
  m.def("gated_feed_forward", &gated_feed_forward);
  m.def("grad_norm", &grad_norm);
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("clipped_adam", &clipped_adam);
}
