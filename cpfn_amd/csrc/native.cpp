// The host side of the routed residual block's operators and of the gradient lists: argument checks, output allocation, launches on
// torch's current stream and the autograd nodes, over the C ABI of include/cpfn_hip.h.  cpfn_amd/ops.py, autograd_ops.py and optim.py
// are its callers.  In C++ because these calls come one after the other from an eager training loop whose kernels take 5 to 80 us:
// as Python functions over ctypes, a forward and backward pass of one operator cost the host 60 to 120 us.
//
// Errors are std::runtime_error (RuntimeError in Python) with the text alone.  Backward passes run on the autograd engine's thread,
// without the interpreter.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <cmath>

#include "../../include/cpfn_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

template <typename... A> [[noreturn]] void fail(const A &...a) { throw std::runtime_error(c10::str(a...)); }
#define REQUIRE(cond, ...)               \
  do {                                   \
    if (!(cond)) fail(__VA_ARGS__);      \
  } while (0)

void check_status(int status, const char *what) {
  if (status == 0) return;
  fail(what, " failed with status ", status,
       status == CPFN_EINVAL ? " (invalid argument)"
       : status == CPFN_EOVERLAP ? " (a tensor that is written shares memory with another one of the lists: a gradient listed twice?)"
                                 : " (hipError_t)");
}

// Algorithmic bytes of a launch for lib.py's counters: a callable (name, bytes) while somebody counts, else nothing.
std::atomic<PyObject *> counter{nullptr};
void set_counter(const py::object &f) {
  PyObject *next = f.is_none() ? nullptr : py::object(f).release().ptr();
  PyObject *old = counter.exchange(next);
  Py_XDECREF(old);
}
void count(const char *name, int64_t bytes) {
  if (!counter.load(std::memory_order_relaxed)) return;
  py::gil_scoped_acquire gil;
  PyObject *f = counter.load();
  if (f) py::reinterpret_borrow<py::object>(f)(name, bytes);
}

Tensor or_none(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *fptr(const Tensor &t) { return (float *)ptr(t); }
void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

int code_of(at::ScalarType t) { return t == at::kFloat ? CPFN_F32 : t == at::kBFloat16 ? CPFN_BF16 : t == at::kHalf ? CPFN_F16 : -1; }

void check_rows(const Tensor &t, const char *name, const Tensor *like = nullptr) {
  REQUIRE(t.is_cuda(), name, " must be a CUDA(HIP) tensor: CPU not supported");
  REQUIRE(t.layout() == at::kStrided && t.dim() == 2 && t.is_contiguous(), name, " must be contiguous rows [P, C]");
  REQUIRE(code_of(t.scalar_type()) >= 0, name, " must be a float32, bfloat16 or float16 tensor");
  if (like)
    REQUIRE(t.scalar_type() == like->scalar_type() && t.device() == like->device(), name,
            " must have the type and the device of the rows it goes with (", like->scalar_type(), " on ", like->device(), ")");
}
void check_vector(const Tensor &t, const char *name, const Tensor &x) {
  if (!t.defined()) return;
  REQUIRE(t.is_cuda(), name, " must be a CUDA(HIP) tensor: CPU not supported");
  REQUIRE(t.scalar_type() == at::kFloat, name, " must be a float32 tensor");
  REQUIRE(t.layout() == at::kStrided && t.dim() == 1 && t.is_contiguous() && t.size(0) == x.size(1) && t.device() == x.device(), name,
          " must hold one value for each of the ", x.size(1), " channels, contiguous, on the rows' device");
}

// ---------------------------------------------------------------- norms around a residual block
constexpr int64_t NORM_MAX_CHANNELS = 4096;

struct Norm {
  Tensor x, y, weight, bias, gate, scale, next_weight, next_bias;
  bool sigmoid, layer;
  double eps;

  void check() const {
    check_rows(x, "x");
    const int64_t P = x.size(0), C = x.size(1);
    REQUIRE(C >= 1 && C <= NORM_MAX_CHANNELS, "norms take 1 to ", NORM_MAX_CHANNELS, " channels (got ", C, ")");
    REQUIRE(eps >= 0.0 && std::isfinite((float)eps), "eps must be finite and not negative");
    if (y.defined()) {
      check_rows(y, "y", &x);
      REQUIRE(y.sizes() == x.sizes(), "y must have the shape of x (got ", y.sizes(), " for ", x.sizes(), ")");
    }
    if (gate.defined()) {
      check_rows(gate, "gate", &x);
      const int64_t G = gate.size(0);
      REQUIRE(gate.size(1) == C && (P == 0 || (G >= 1 && P % G == 0)),
              "gate must be [P, C], or [G, C] for G groups of P / G consecutive rows (got ", gate.sizes(), " for ", x.sizes(), ")");
    }
    check_vector(weight, "weight", x);
    check_vector(bias, "bias", x);
    check_vector(scale, "scale", x);
    check_vector(next_weight, "next_weight", x);
    check_vector(next_bias, "next_bias", x);
    REQUIRE(!bias.defined() || weight.defined(), "a bias needs its weight (no weight: no norm)");
    REQUIRE(!next_bias.defined() || next_weight.defined(), "next_bias needs next_weight (no next_weight: no norm)");
    REQUIRE(y.defined() || (!weight.defined() && !gate.defined() && !scale.defined() && next_weight.defined()),
            "without y there is only the norm of x: next_weight, next_bias");
  }
  int64_t gate_rows() const { return gate.defined() ? gate.size(0) : 0; }
  int64_t gate_values() const { return gate.defined() ? gate.numel() : 0; }

  std::pair<Tensor, Tensor> forward() const {
    check();
    const int64_t P = x.size(0), C = x.size(1);
    Tensor out, normed;
    if (y.defined()) out = at::empty({P, C}, x.options());
    if (next_weight.defined()) normed = at::empty({P, C}, x.options());
    if (P == 0) return {out, normed};
    const c10::DeviceGuard guard(x.device());
    check_status(cpfn_norm_residual_fwd(ptr(x), ptr(y), ptr(gate), fptr(weight), fptr(bias), fptr(scale), fptr(next_weight),
                                        fptr(next_bias), P, (int)C, gate_rows(), code_of(x.scalar_type()), layer, sigmoid, (float)eps, ptr(out),
                                        ptr(normed), stream_of(x)),
                 "cpfn_norm_residual_fwd");
    count("cpfn_norm_residual_fwd", x.element_size() * (P * C * (1 + 2 * y.defined() + normed.defined()) + gate_values()));
    return {out, normed};
  }

  // gradients of x, y, weight, bias, gate, scale, next_weight, next_bias, as `needs` asks for them
  std::array<Tensor, 8> backward(const Tensor &d_out, const Tensor &d_normed, std::array<bool, 8> needs) const {
    check();
    for (const auto &[t, name] : {std::pair<const Tensor &, const char *>{d_out, "d_out"}, {d_normed, "d_normed"}})
      if (t.defined()) {
        check_rows(t, name, &x);
        REQUIRE(t.sizes() == x.sizes(), name, " must have the shape of x");
      }
    REQUIRE(d_out.defined() || d_normed.defined(), "no gradient: d_out and d_normed are both None");
    REQUIRE(!d_normed.defined() || next_weight.defined(), "d_normed needs next_weight");
    const int64_t P = x.size(0), C = x.size(1);
    const bool given[8] = {true, y.defined(), weight.defined(), bias.defined(), gate.defined(), scale.defined(), d_normed.defined(), d_normed.defined()};
    std::array<Tensor, 8> g;
    bool any = false;
    for (int i = 0; i < 8; ++i) any |= needs[i] &= given[i];
    if (!any) return g;
    for (int i : {0, 1})
      if (needs[i]) g[i] = at::empty({P, C}, x.options());
    if (needs[4]) g[4] = P == 0 ? at::zeros(gate.sizes(), x.options()) : at::empty(gate.sizes(), x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    for (int i : {2, 3, 5, 6, 7})
      if (needs[i]) g[i] = P == 0 ? at::zeros({C}, f32) : at::empty({C}, f32);
    if (P == 0) return g;
    const c10::DeviceGuard guard(x.device());
    const Tensor ws = at::empty({cpfn_norm_residual_workspace(P, (int)C, gate_rows()) / 4}, f32);
    check_status(cpfn_norm_residual_bwd(ptr(x), ptr(y), ptr(gate), fptr(weight), fptr(bias), fptr(scale), fptr(next_weight), ptr(d_out),
                                        ptr(d_normed), P, (int)C, gate_rows(), code_of(x.scalar_type()), layer, sigmoid, (float)eps, ptr(g[0]),
                                        ptr(g[1]), ptr(g[4]), fptr(g[2]), fptr(g[3]), fptr(g[5]), fptr(g[6]), fptr(g[7]), ptr(ws), stream_of(x)),
                 "cpfn_norm_residual_bwd");
    count("cpfn_norm_residual_bwd",
          x.element_size() * (P * C * (y.defined() + d_out.defined() + 2 * d_normed.defined() + g[0].defined() + g[1].defined()) +
                              gate_values() * (1 + g[4].defined())));
    return g;
  }
};

std::tuple<Maybe, Maybe> pair_of(const Tensor &a, const Tensor &b) {
  return {a.defined() ? Maybe(a) : std::nullopt, b.defined() ? Maybe(b) : std::nullopt};
}

std::tuple<Maybe, Maybe> norm_residual_fwd(const Tensor &x, const Maybe &y, const Maybe &weight, const Maybe &bias, const Maybe &gate, bool sigmoid,
                                           const Maybe &scale, const Maybe &next_weight, const Maybe &next_bias, bool layer, double eps) {
  const auto r = Norm{x, or_none(y), or_none(weight), or_none(bias), or_none(gate), or_none(scale), or_none(next_weight), or_none(next_bias), sigmoid, layer, eps}.forward();
  return pair_of(r.first, r.second);
}
std::vector<Maybe> norm_residual_bwd(const Tensor &x, const Maybe &y, const Maybe &weight, const Maybe &bias, const Maybe &gate, bool sigmoid,
                                     const Maybe &scale, const Maybe &next_weight, const Maybe &d_out, const Maybe &d_normed, bool layer, double eps,
                                     std::array<bool, 8> needs) {
  const auto g = Norm{x, or_none(y), or_none(weight), or_none(bias), or_none(gate), or_none(scale), or_none(next_weight), Tensor(), sigmoid, layer, eps}.backward(
      or_none(d_out), or_none(d_normed), needs);
  std::vector<Maybe> r;
  for (const Tensor &t : g) r.push_back(t.defined() ? Maybe(t) : std::nullopt);
  return r;
}

// Results that can be used, but not differentiated: autograd raises `error` where it comes to them.
void not_differentiable(variable_list &results, std::string error) {
  variable_list in;
  for (Tensor &g : results)
    if (g.defined()) {
      in.push_back(g.detach());
      in.back().set_requires_grad(true);
    }
  if (in.empty()) return;
  auto node = std::make_shared<torch::autograd::DelayedError>(std::move(error), (int64_t)in.size());
  auto out = (*node)(std::move(in));
  size_t k = 0;
  for (Tensor &g : results)
    if (g.defined()) g = out[k++];
}
// The gradients of a backward pass that is itself recorded (create_graph).
void not_again(variable_list &grads, const char *what) {
  if (at::GradMode::is_enabled()) not_differentiable(grads, c10::str(what, " is differentiable once: its gradients cannot be differentiated"));
}

// Forward-mode derivatives (torch.autograd.forward_ad) are refused: a kernel reads an input's value alone, and its result would stand for
// one whose derivative is zero.  Also where autograd records nothing: neither requires_grad nor no_grad says anything about them.  There
// are tangents only while a dual level is open, which is asked first (tensor by tensor a list of 301 cost 2 us more).
bool tangents_about() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
bool tangent(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
bool tangent(const Maybe &t) { return t.has_value() && tangent(*t); }
template <typename... A> void refuse_tangents(const char *what, const A &...tensors) {
  REQUIRE(!tangents_about() || !(tangent(tensors) || ...), what,
          " has no forward-mode derivative (a tensor carries a tangent: torch.autograd.forward_ad.unpack_dual gives its value)");
}

// A backward pass that is captured must not reach a leaf whose gradient is accumulated on the default stream, which cannot take part in a
// capture.  It is where an eager graph of the same leaf, built on that stream, is still alive: the leaf has one accumulating node, which
// keeps the stream that it was made on.
void check_capture(const Tensor &on) {
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(on.get_device());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (stream.stream() == nullptr || hipStreamIsCapturing(stream.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto &edge : node->next_edges()) {
    if (!dynamic_cast<torch::autograd::AccumulateGrad *>(edge.function.get())) continue;
    const auto made_on = edge.function->stream();
    REQUIRE(!made_on || c10::hip::HIPStreamMasqueradingAsCUDA(*made_on).stream() != nullptr,
            "a backward pass is captured while an eager graph of the same leaf lives on the default stream: drop that graph's results first");
  }
}

// Does autograd record this call?  (A node costs a call of 5 us another one where nobody asks for it.)
template <typename... A> bool recorded(const A &...tensors) { return at::GradMode::is_enabled() && (or_none(tensors).requires_grad() || ...); }

Tensor contiguous(const Tensor &t) { return t.defined() ? t.contiguous() : t; }

// The end of a residual block and the norm of the next one as one node.  Only the inputs are kept: out, the normalised rows and both
// norms' statistics are formed again from them, in fp32 as the forward pass had them.
struct NormResidual : public torch::autograd::Function<NormResidual> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &y, const Maybe &weight, const Maybe &bias, const Maybe &gate,
                               const Maybe &scale, const Maybe &next_weight, const Maybe &next_bias, bool sigmoid, bool layer, double eps) {
    const Norm n{x.contiguous(), contiguous(or_none(y)), or_none(weight), or_none(bias), contiguous(or_none(gate)), or_none(scale), or_none(next_weight),
                 or_none(next_bias), sigmoid, layer, eps};
    const auto r = n.forward();
    ctx->save_for_backward({n.x, n.y, n.weight, n.bias, n.gate, n.scale, n.next_weight});
    ctx->set_materialize_grads(false);
    ctx->saved_data["how"] = (int64_t)(sigmoid | layer << 1 | n.next_bias.defined() << 2);
    ctx->saved_data["eps"] = eps;
    variable_list out;
    for (const Tensor &t : {r.first, r.second})
      if (t.defined()) out.push_back(t);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &d) {
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    for (const Tensor &t : d) refuse_tangents("norm_residual", t);
    const int64_t how = ctx->saved_data["how"].toInt();
    const Norm n{saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], Tensor(), (how & 1) != 0, (how & 2) != 0, ctx->saved_data["eps"].toDouble()};
    const bool given[8] = {true, n.y.defined(), n.weight.defined(), n.bias.defined(), n.gate.defined(), n.scale.defined(), n.next_weight.defined(), (how & 4) != 0};
    std::array<bool, 8> needs{};
    size_t edge = 0;
    for (int i = 0; i < 8; ++i)
      if (given[i]) needs[i] = ctx->needs_input_grad(edge++);
    size_t k = 0;
    const Tensor d_out = n.y.defined() ? contiguous(d[k++]) : Tensor(), d_normed = k < d.size() ? contiguous(d[k]) : Tensor();
    variable_list grads(11);
    if (d_out.defined() || d_normed.defined()) {
      const auto g = n.backward(d_out, d_normed, needs);
      for (int i = 0; i < 8; ++i) grads[i] = g[i];
    }
    not_again(grads, "norm_residual");
    return grads;
  }
};

std::tuple<Maybe, Maybe> norm_residual(const Tensor &x, const Maybe &y, const Maybe &weight, const Maybe &bias, const Maybe &gate, bool sigmoid,
                                       const Maybe &scale, const Maybe &next_weight, const Maybe &next_bias, bool layer, double eps) {
  refuse_tangents("norm_residual", x, y, weight, bias, gate, scale, next_weight, next_bias);
  if (!recorded(x, y, weight, bias, gate, scale, next_weight, next_bias)) {
    const auto r = Norm{x.contiguous(), contiguous(or_none(y)), or_none(weight), or_none(bias), contiguous(or_none(gate)), or_none(scale), or_none(next_weight),
                        or_none(next_bias), sigmoid, layer, eps}.forward();
    return pair_of(r.first, r.second);
  }
  const auto r = NormResidual::apply(x, y, weight, bias, gate, scale, next_weight, next_bias, sigmoid, layer, eps);
  return pair_of(y.has_value() ? r[0] : Tensor(), next_weight.has_value() ? r.back() : Tensor());
}

// ---------------------------------------------------------------- rows sorted by expert and back
constexpr int64_t ROUTE_MAX_EXPERTS = 2048, ROUTE_MAX_CHANNELS = 1ll << 30;

std::tuple<Tensor, Tensor> route_plan(const Tensor &choice, int64_t E) {
  REQUIRE(choice.is_cuda(), "choice must be a CUDA(HIP) tensor: CPU not supported");
  REQUIRE(choice.layout() == at::kStrided && choice.dim() == 2 && choice.is_contiguous(), "choice must be contiguous [R, k]");
  const bool wide = choice.scalar_type() == at::kLong;
  REQUIRE(wide || choice.scalar_type() == at::kInt, "choice must be an int32 or int64 tensor");
  REQUIRE(E >= 1 && E <= ROUTE_MAX_EXPERTS, "routing takes 1 to ", ROUTE_MAX_EXPERTS, " experts (got ", E, ")");
  const int64_t n = choice.numel();
  REQUIRE(choice.size(1) >= 1 && n < (1ll << 31), "choice must hold at least one choice for each row and fewer than 2^31 in all (got ", choice.sizes(), ")");
  const auto i32 = choice.options().dtype(at::kInt);
  Tensor offsets = at::empty({E + 1}, i32), place = at::empty(choice.sizes(), i32), ws;
  const c10::DeviceGuard guard(choice.device());
  if (const long long bytes = cpfn_route_workspace(n, (int)E)) ws = at::empty({bytes / 4}, i32);
  check_status(cpfn_route_plan(ptr(choice), wide, n, (int)E, (int *)ptr(offsets), (int *)ptr(place), ptr(ws), stream_of(choice)), "cpfn_route_plan");
  count("cpfn_route_plan", (choice.element_size() + 4) * n + 4 * (E + 1));
  return {offsets, place};
}

struct Plan {
  Tensor offsets, place;
  int64_t E;
  int64_t R() const { return place.size(0); }
  int64_t k() const { return place.size(1); }
  void check(const Tensor &t, const char *name, bool sorted) const {
    REQUIRE(place.is_cuda() && place.scalar_type() == at::kInt && place.dim() == 2 && place.is_contiguous() && offsets.scalar_type() == at::kInt &&
                offsets.dim() == 1 && offsets.is_contiguous() && offsets.size(0) == E + 1 && offsets.device() == place.device(),
            "plan must be a RoutePlan of ops.route_plan");
    check_rows(t, name);
    const int64_t rows = sorted ? R() * k() : R();
    REQUIRE(t.size(0) == rows && t.device() == place.device(), name, " must have ", rows, " rows, on the plan's device (got ", t.sizes(), ")");
    REQUIRE(t.size(1) >= 1 && t.size(1) <= ROUTE_MAX_CHANNELS, name, " must have 1 to 2^30 channels (got ", t.size(1), ")");
  }
  void check_weights(const Tensor &w) const {
    if (!w.defined()) return;
    REQUIRE(w.is_cuda(), "weights must be a CUDA(HIP) tensor: CPU not supported");
    REQUIRE(w.scalar_type() == at::kFloat && w.layout() == at::kStrided && w.is_contiguous() && w.sizes() == place.sizes() && w.device() == place.device(),
            "weights must be contiguous float32 [R, k] = ", place.sizes(), ", on the plan's device");
  }
};

Tensor gather_rows(const Tensor &rows, const Plan &p) {
  p.check(rows, "rows", false);
  const int64_t R = p.R(), k = p.k(), C = rows.size(1);
  Tensor out = at::empty({R * k, C}, rows.options());
  if (R == 0) return out;
  const c10::DeviceGuard guard(rows.device());
  check_status(cpfn_route_gather(ptr(rows), (int *)ptr(p.place), (int *)ptr(p.offsets), R, (int)k, (int)p.E, (int)C, code_of(rows.scalar_type()), ptr(out),
                                 stream_of(rows)),
               "cpfn_route_gather");
  count("cpfn_route_gather", rows.element_size() * (R + R * k) * C + 4 * R * k);
  return out;
}
Tensor combine_rows(const Tensor &sorted, const Tensor &weights, const Plan &p) {
  p.check(sorted, "sorted_rows", true);
  p.check_weights(weights);
  const int64_t R = p.R(), k = p.k(), C = sorted.size(1);
  Tensor out = at::empty({R, C}, sorted.options());
  if (R == 0) return out;
  const c10::DeviceGuard guard(sorted.device());
  check_status(cpfn_route_combine(ptr(sorted), fptr(weights), (int *)ptr(p.place), R, (int)k, (int)C, code_of(sorted.scalar_type()), ptr(out), stream_of(sorted)),
               "cpfn_route_combine");
  count("cpfn_route_combine", sorted.element_size() * (R + R * k) * C + (weights.defined() ? 8 : 4) * R * k);
  return out;
}
std::pair<Tensor, Tensor> combine_rows_bwd(const Tensor &g, const Tensor &sorted, const Tensor &weights, const Plan &p, bool need_rows, bool need_weights) {
  p.check(g, "grad_out", false);
  p.check_weights(weights);
  const int64_t R = p.R(), k = p.k(), C = g.size(1);
  Tensor d_sorted, d_weights;
  if (!need_rows && !need_weights) return {d_sorted, d_weights};
  if (need_weights) {
    REQUIRE(sorted.defined(), "the weights' gradient needs sorted_rows");
    p.check(sorted, "sorted_rows", true);
    check_rows(sorted, "sorted_rows", &g);
    REQUIRE(sorted.size(1) == C, "sorted_rows and grad_out must have the same channels");
    d_weights = at::empty({R, k}, g.options().dtype(at::kFloat));
  }
  if (need_rows) d_sorted = at::empty({R * k, C}, g.options());
  if (R == 0) return {d_sorted, d_weights};
  const c10::DeviceGuard guard(g.device());
  check_status(cpfn_route_combine_bwd(ptr(g), need_weights ? ptr(sorted) : nullptr, fptr(weights), (int *)ptr(p.place), (int *)ptr(p.offsets), R, (int)k,
                                      (int)p.E, (int)C, code_of(g.scalar_type()), ptr(d_sorted), fptr(d_weights), stream_of(g)),
               "cpfn_route_combine_bwd");
  count("cpfn_route_combine_bwd", g.element_size() * (R + R * k * (need_rows + need_weights)) * C + 12 * R * k);
  return {d_sorted, d_weights};
}

struct RouteGather : public torch::autograd::Function<RouteGather> {
  static Tensor forward(AutogradContext *ctx, const Tensor &rows, const Tensor &offsets, const Tensor &place, int64_t E) {
    ctx->save_for_backward({offsets, place});
    ctx->saved_data["E"] = E;
    return gather_rows(rows.contiguous(), Plan{offsets, place, E});
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &d) {
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[1]);
    refuse_tangents("route_gather", d[0]);
    variable_list grads(4);
    grads[0] = combine_rows(d[0].contiguous(), Tensor(), Plan{saved[0], saved[1], ctx->saved_data["E"].toInt()});
    not_again(grads, "route_gather");
    return grads;
  }
};
struct RouteCombine : public torch::autograd::Function<RouteCombine> {
  static Tensor forward(AutogradContext *ctx, const Tensor &sorted_, const Maybe &weights_, const Tensor &offsets, const Tensor &place, int64_t E) {
    const Tensor sorted = sorted_.contiguous(), weights = contiguous(or_none(weights_));
    ctx->save_for_backward({weights.defined() && weights_->requires_grad() ? sorted : Tensor(), weights, offsets, place});
    ctx->saved_data["E"] = E;
    return combine_rows(sorted, weights, Plan{offsets, place, E});
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &d) {
    const auto saved = ctx->get_saved_variables();
    check_capture(saved[3]);
    refuse_tangents("route_combine", d[0]);
    const bool weighted = saved[1].defined();
    const auto g = combine_rows_bwd(d[0].contiguous(), saved[0], saved[1], Plan{saved[2], saved[3], ctx->saved_data["E"].toInt()}, ctx->needs_input_grad(0),
                                    weighted && ctx->needs_input_grad(1));
    variable_list grads(5);
    grads[0] = g.first;
    grads[1] = g.second;
    not_again(grads, "route_combine");
    return grads;
  }
};

// ---------------------------------------------------------------- lists of gradients
// elements fill one stretch of memory, in whatever order of the dimensions
bool dense(const Tensor &t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

struct Table {
  std::vector<void *> at;
  std::vector<long long> n;
  std::vector<int> type;
  int64_t bytes = 0;
  bool recorded = false;                     // a tensor that autograd follows
  const bool tangents = tangents_about();

  const Tensor &add(PyObject *o, const char *name, c10::Device &device) {
    REQUIRE(THPVariable_Check(o), name, " must be tensors");
    const Tensor &t = THPVariable_Unpack(o);
    if (tangents) refuse_tangents(name, t);
    recorded |= t.requires_grad();
    REQUIRE(t.is_cuda(), name, " must be CUDA(HIP) tensors: CPU not supported");
    if (device.is_cpu()) device = t.device();
    REQUIRE(t.device() == device, name, " must be on one device (got ", device, " and ", t.device(), ")");
    const int code = code_of(t.scalar_type());
    REQUIRE(code >= 0, name, " must be float32, bfloat16 or float16 tensors (got ", t.scalar_type(), ")");
    REQUIRE(t.layout() == at::kStrided && dense(t), name, " must be dense and without overlap");
    at.push_back(t.data_ptr());
    n.push_back(t.numel());
    type.push_back(code);
    bytes += t.numel() * t.element_size();
    return t;
  }
};

// the norm over all gradients; max_norm: clipped to it, in place or into `out`.  The norm of tensors that autograd follows (gradients of
// create_graph, parameters) has a value and no derivative: differentiating it raises.  Clipping works on values, as under no_grad.
Tensor grad_norm(const py::list &grads, int p, std::optional<double> max_norm, const std::optional<py::list> &out) {
  const size_t count_ = grads.size();
  REQUIRE(!out || out->size() == count_, "out must have a tensor for each gradient (got ", out ? out->size() : 0, " for ", count_, ")");
  if (max_norm) REQUIRE(*max_norm >= 0.0, "max_norm must not be negative (got ", *max_norm, ")");
  if (count_ == 0) return at::zeros({});
  c10::Device device(at::kCPU);
  Table src, dst;
  for (size_t i = 0; i < count_; ++i) {
    const Tensor &g = src.add(PyList_GET_ITEM(grads.ptr(), i), "grads", device);
    if (!out) continue;
    const Tensor &o = dst.add(PyList_GET_ITEM(out->ptr(), i), "out", device);
    REQUIRE(o.sizes() == g.sizes() && (o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous())),
            "out must have the gradients' shapes and order of dimensions (got ", o.sizes(), " for ", g.sizes(), ")");
    REQUIRE(o.scalar_type() == g.scalar_type() || o.scalar_type() == at::kFloat, "out must be of the gradient's type or float32 (got ", o.scalar_type(), " for ",
            g.scalar_type(), ")");
  }
  const c10::DeviceGuard guard(device);
  const auto options = at::TensorOptions().device(device);
  const Tensor norm = at::empty({}, options.dtype(at::kFloat));
  const Tensor ws = at::empty({cpfn_grad_norm_workspace(src.n.data(), (int)count_) / 8}, options.dtype(at::kDouble));
  void *stream = stream_of(norm);
  if (max_norm) {
    check_status(cpfn_grad_clip(src.at.data(), out ? dst.at.data() : nullptr, src.n.data(), src.type.data(), out ? dst.type.data() : nullptr, (int)count_, p,
                                *max_norm, fptr(norm), ptr(ws), stream),
                 "cpfn_grad_clip");
    for (size_t i = 0; i < count_; ++i) {                 // (written behind autograd's back)
      const Tensor &t = THPVariable_Unpack(PyList_GET_ITEM(out ? out->ptr() : grads.ptr(), i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
    count("cpfn_grad_clip", src.bytes + (out ? dst.bytes : src.bytes));
  } else {
    check_status(cpfn_grad_norm(src.at.data(), src.n.data(), src.type.data(), (int)count_, p, fptr(norm), ptr(ws), stream), "cpfn_grad_norm");
    count("cpfn_grad_norm", src.bytes);
    if (src.recorded && at::GradMode::is_enabled()) {
      variable_list r{norm};
      not_differentiable(r, "grad_norm has no derivative: under torch.no_grad(), or of detached tensors, it is a plain value");
      return r[0];
    }
  }
  return norm;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  typedef py::call_guard<py::gil_scoped_release> free_gil;
  m.def("set_counter", &set_counter);
  m.def("norm_residual_fwd", &norm_residual_fwd, free_gil());
  m.def("norm_residual_bwd", &norm_residual_bwd, free_gil());
  m.def("norm_residual", &norm_residual, free_gil());
  m.def("route_plan", &route_plan, free_gil());
  m.def("route_gather_fwd", [](const Tensor &rows, const Tensor &offsets, const Tensor &place, int64_t E) { return gather_rows(rows, Plan{offsets, place, E}); }, free_gil());
  m.def("route_combine_fwd", [](const Tensor &sorted, const Maybe &weights, const Tensor &offsets, const Tensor &place, int64_t E) {
    return combine_rows(sorted, or_none(weights), Plan{offsets, place, E});
  }, free_gil());
  m.def("route_combine_bwd", [](const Tensor &g, const Maybe &sorted, const Maybe &weights, const Tensor &offsets, const Tensor &place, int64_t E, bool need_rows,
                                bool need_weights) {
    const auto r = combine_rows_bwd(g, or_none(sorted), or_none(weights), Plan{offsets, place, E}, need_rows, need_weights);
    return pair_of(r.first, r.second);
  }, free_gil());
  m.def("route_gather", [](const Tensor &rows, const Tensor &offsets, const Tensor &place, int64_t E) {
    refuse_tangents("route_gather", rows);
    return recorded(rows) ? RouteGather::apply(rows, offsets, place, E) : gather_rows(rows.contiguous(), Plan{offsets, place, E});
  }, free_gil());
  m.def("route_combine", [](const Tensor &sorted, const Maybe &weights, const Tensor &offsets, const Tensor &place, int64_t E) {
    refuse_tangents("route_combine", sorted, weights);
    if (!recorded(sorted, weights)) return combine_rows(sorted.contiguous(), contiguous(or_none(weights)), Plan{offsets, place, E});
    return RouteCombine::apply(sorted, weights, offsets, place, E);
  }, free_gil());
  m.def("grad_norm", &grad_norm);
}
