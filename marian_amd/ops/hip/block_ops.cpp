// Entry points of the recurrent block's operators: argument checks and
// autograd in C++. A decode step or a short sequence takes a few microseconds
// on the GPU; checks, allocations and graph nodes in Python took 11 us for a
// step and about 100 us for a training pass, more than the kernels.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "fresh.h"

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::vector<Tensor> gated_scan_fwd(Tensor x, Tensor gate, OptTensor state,
                                   OptTensor lens, bool reverse, bool relu,
                                   bool want_bnd);
Tensor gated_scan_bwd(Tensor x, Tensor gate, OptTensor state, OptTensor lens,
                      Tensor bnd, OptTensor dy, OptTensor dlast, bool reverse,
                      bool relu, Tensor dx, Tensor dgate, bool want_dstate);
Tensor gated_step_fwd(Tensor x, Tensor gate, Tensor state, Tensor state_out,
                      bool relu);
std::vector<Tensor> block_norm_fwd(at::IntArrayRef sizes, Tensor x,
                                   OptTensor res, OptTensor gate,
                                   bool highway, double alpha,
                                   OptTensor post_scale, OptTensor post_bias,
                                   OptTensor pre_scale, OptTensor pre_bias,
                                   bool rms, double eps, bool want_stat);
std::vector<Tensor> block_norm_bwd(
    Tensor x, OptTensor res, OptTensor gate, bool highway, double alpha,
    OptTensor post_scale, OptTensor post_bias, OptTensor pre_scale,
    OptTensor pre_bias, bool rms, double eps, Tensor stat, OptTensor dsum,
    OptTensor dh, std::vector<bool> want);

namespace {

// a refused argument is a ValueError, as it is off the GPU
#define REFUSE_UNLESS(cond, ...) \
  if (!(cond)) throw pybind11::value_error(c10::str(__VA_ARGS__))

OptTensor opt(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}
Tensor plain(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// The kernels are called on memory: a tangent would be dropped and a trace
// would hold the outputs as constants, neither with a word.
template <typename... Ts>
void refuse_modes(const char* what, const Ts&... ts) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !((ts.defined() && ts._fw_grad(0).defined()) || ...), what,
      " has no forward-mode derivative");
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(), what,
                              " cannot be traced on the GPU");
}

bool dtype_ok(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == torch::kFloat32 || s == torch::kBFloat16 || s == torch::kHalf;
}

// The gradients have no gradient of their own: under create_graph they carry
// a node that says so when it is reached.
variable_list once(variable_list outs) {
  if (!c10::GradMode::is_enabled()) return outs;
  auto err = std::make_shared<torch::autograd::DelayedError>(
      "this operator is differentiable once only", (int64_t)outs.size());
  for (auto& t : outs)
    if (t.defined()) t = t.detach().requires_grad_();
  return (*err)(std::move(outs));
}

// ---- gated linear recurrence ----------------------------------------------

bool act_relu(const char* what, const std::string& act) {
  REFUSE_UNLESS(act == "none" || act == "relu", what,
                ": act must be one of ('none', 'relu'), got '", act, "'");
  return act == "relu";
}

void check_scan(const char* what, const Tensor& x, const Tensor& gate,
                const Tensor& state, const Tensor& lens, int64_t dims) {
  REFUSE_UNLESS(x.dim() == dims, what, ": x must have ", dims,
                " dimensions, got ", x.sizes());
  REFUSE_UNLESS(gate.sizes() == x.sizes(), what, ": gate ", gate.sizes(),
                " must have x's shape ", x.sizes());
  REFUSE_UNLESS(gate.scalar_type() == x.scalar_type() &&
                    gate.device() == x.device(),
                what, ": x and gate must share dtype and device");
  // a fused projection's rows are twice as wide; lane offsets reach 2^26
  REFUSE_UNLESS(x.size(-1) > 0 && x.size(-1) < (1L << 25), what,
                ": the width must be 1..2^25-1, got ", x.size(-1));
  REFUSE_UNLESS(dtype_ok(x), what, ": unsupported dtype ", x.scalar_type());
  if (state.defined())
    REFUSE_UNLESS(state.dim() == 2 && state.size(0) == x.size(0) &&
                      state.size(1) == x.size(-1) &&
                      state.scalar_type() == torch::kFloat32 &&
                      state.device() == x.device(),
                  what, ": state must be float32 [", x.size(0), ", ",
                  x.size(-1), "] on x's device");
  if (lens.defined())
    REFUSE_UNLESS(lens.dim() == 1 && lens.size(0) == x.size(0) &&
                      lens.scalar_type() == torch::kInt32 &&
                      lens.device() == x.device(),
                  what, ": lens must be int32 [", x.size(0),
                  "] on x's device");
}

// t, or a copy if its last dimension is not dense or its rows lie further
// apart than the kernels' 32-bit lane offsets reach
Tensor dense_rows(const Tensor& t) {
  if (t.size(-1) != 1 && t.stride(-1) != 1) return t.contiguous();
  if (t.dim() == 3 && t.size(1) > 1 && t.stride(1) >= (1L << 26))
    return t.contiguous();
  return t;
}

Tensor half(const Tensor& xg, int which) {
  const int64_t d = xg.size(-1) / 2;
  return xg.narrow(-1, which * d, d);
}

// gate undefined: x is the fused projection [B, T, 2D], read in place, whose
// gradient comes out as one buffer
struct ScanFn : public torch::autograd::Function<ScanFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const OptTensor& gate, const OptTensor& state,
                               const OptTensor& lens, bool reverse,
                               bool relu) {
    const bool fused = !gate.has_value();
    auto out = gated_scan_fwd(fused ? half(x, 0) : x,
                              fused ? half(x, 1) : *gate, state, lens, reverse,
                              relu, true);
    ctx->save_for_backward({x, plain(gate), plain(state), plain(lens),
                            out[2]});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["relu"] = relu;
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const bool fused = !s[1].defined();
    // absent inputs have no edge
    const bool want_state =
        s[2].defined() && ctx->needs_input_grad(fused ? 1 : 2);
    Tensor dx = mamd::fresh_like(s[0]);
    Tensor dg = fused ? Tensor() : mamd::fresh_like(s[0]);
    auto ds = gated_scan_bwd(
        fused ? half(s[0], 0) : s[0], fused ? half(s[0], 1) : s[1], opt(s[2]),
        opt(s[3]), s[4], opt(g[0]),
        g[1].defined() ? OptTensor(g[1].contiguous()) : OptTensor(),
        ctx->saved_data["reverse"].toBool(), ctx->saved_data["relu"].toBool(),
        fused ? half(dx, 0) : dx, fused ? half(dx, 1) : dg, want_state);
    return once({dx, dg, ds, Tensor(), Tensor(), Tensor()});
  }
};

std::tuple<Tensor, Tensor> scan(Tensor x, Tensor gate, Tensor state,
                                Tensor lens, bool reverse, bool relu) {
  x = dense_rows(x);
  if (gate.defined()) gate = dense_rows(gate);
  if (state.defined()) state = state.contiguous();
  if (lens.defined()) lens = lens.contiguous();
  if (c10::GradMode::is_enabled() &&
      (wants_grad(x) || wants_grad(gate) || wants_grad(state))) {
    auto out = ScanFn::apply(x, opt(gate), opt(state), opt(lens), reverse,
                             relu);
    return {out[0], out[1]};
  }
  const bool fused = !gate.defined();
  auto out = gated_scan_fwd(fused ? half(x, 0) : x, fused ? half(x, 1) : gate,
                            opt(state), opt(lens), reverse, relu, false);
  return {out[0], out[1]};
}

// ---- block join -----------------------------------------------------------

// [R, D] of a dense tensor; without a graph node when called in a Function
Tensor rows(const Tensor& t) {
  return t.dim() == 2 ? t : t.view({t.numel() / t.size(-1), t.size(-1)});
}
// the other way round
Tensor like(const Tensor& rows, const Tensor& t) {
  return t.dim() == rows.dim() ? rows : rows.view(t.sizes());
}
OptTensor rows(const OptTensor& t, bool channel) {
  return !t.has_value() || channel ? t : OptTensor(rows(*t));
}

// x, res (or none) and a per-token gate: dense, of one shape
struct JoinFn : public torch::autograd::Function<JoinFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x,
                               const OptTensor& res, const OptTensor& gate,
                               const OptTensor& w1, const OptTensor& b1,
                               const OptTensor& w2, const OptTensor& b2,
                               bool channel, bool highway, double alpha,
                               bool rms, double eps) {
    auto out = block_norm_fwd(x.sizes(), rows(x), rows(res, false),
                              rows(gate, channel), highway, alpha, w1, b1, w2,
                              b2, rms, eps, true);
    ctx->save_for_backward({x, plain(res), plain(gate), plain(w1), plain(b1),
                            plain(w2), plain(b2), out[2]});
    ctx->saved_data["channel"] = channel;
    ctx->saved_data["highway"] = highway;
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    // not views of rows: a caller may change them in place
    if (!w2.has_value()) return {out[0]};
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    std::vector<bool> want(7);
    size_t edge = 0;  // absent inputs have none
    for (size_t i = 0; i < 7; ++i)
      want[i] = s[i].defined() && ctx->needs_input_grad(edge++);
    const bool channel = ctx->saved_data["channel"].toBool();
    auto grad = [&](size_t i) {
      return i < g.size() && g[i].defined() ? OptTensor(rows(g[i].contiguous()))
                                            : OptTensor();
    };
    auto out = block_norm_bwd(
        rows(s[0]), rows(opt(s[1]), false), rows(opt(s[2]), channel),
        ctx->saved_data["highway"].toBool(),
        ctx->saved_data["alpha"].toDouble(), opt(s[3]), opt(s[4]), opt(s[5]),
        opt(s[6]), ctx->saved_data["rms"].toBool(),
        ctx->saved_data["eps"].toDouble(), s[7], grad(0), grad(1), want);
    for (size_t i = 0; i < 3; ++i)
      if (out[i].defined()) out[i] = like(out[i], s[i]);
    out.resize(12);
    return once(std::move(out));
  }
};

}  // namespace

std::tuple<Tensor, Tensor> gated_scan(Tensor x, Tensor gate, OptTensor state,
                                      OptTensor lens, bool reverse,
                                      std::string act) {
  refuse_modes("gated_scan", x, gate, plain(state));
  check_scan("gated_scan", x, gate, plain(state), plain(lens), 3);
  return scan(x, gate, plain(state), plain(lens), reverse,
              act_relu("gated_scan", act));
}

std::tuple<Tensor, Tensor> gated_scan_xg(Tensor xg, OptTensor state,
                                         OptTensor lens, bool reverse,
                                         std::string act) {
  refuse_modes("gated_scan_xg", xg, plain(state));
  REFUSE_UNLESS(xg.dim() == 3 && xg.size(-1) % 2 == 0,
                "gated_scan_xg: xg must be [B, T, 2D], got ", xg.sizes());
  const Tensor x = half(xg, 0);
  check_scan("gated_scan_xg", x, x, plain(state), plain(lens), 3);
  return scan(xg, Tensor(), plain(state), plain(lens), reverse,
              act_relu("gated_scan_xg", act));
}

std::tuple<Tensor, Tensor> gated_step(Tensor x, Tensor gate, OptTensor state_,
                                      std::string act, bool inplace) {
  REFUSE_UNLESS(state_.has_value(), "gated_step: state is required");
  Tensor state = *state_;
  refuse_modes("gated_step", x, gate, state);
  check_scan("gated_step", x, gate, state, Tensor(), 2);
  const bool relu = act_relu("gated_step", act);
  const bool grad = c10::GradMode::is_enabled() &&
                    (wants_grad(x) || wants_grad(gate) || wants_grad(state));
  if (inplace) {
    REFUSE_UNLESS(!grad, "gated_step: inplace has no gradient");
    REFUSE_UNLESS(state.is_contiguous(),
                  "gated_step: inplace needs a dense state");
    REFUSE_UNLESS(!state.is_alias_of(x) && !state.is_alias_of(gate),
                  "gated_step: inplace needs a state of its own memory");
  } else if (grad) {
    auto out = scan(x.unsqueeze(1), gate.unsqueeze(1), state, Tensor(), false,
                    relu);
    return {std::get<0>(out).squeeze(1), std::get<1>(out)};
  }
  state = state.contiguous();
  Tensor out = inplace ? state : mamd::fresh_like(state);
  Tensor y = gated_step_fwd(dense_rows(x), dense_rows(gate), state, out, relu);
  // a graph that saved the old state must notice
  if (inplace && !state.is_inference()) torch::autograd::impl::bump_version(state);
  return {y, out};
}

std::tuple<Tensor, OptTensor> block_norm(
    Tensor x, OptTensor res_, OptTensor gate_, std::string gate_kind, double alpha,
    OptTensor post_scale, OptTensor post_bias, OptTensor pre_scale,
    OptTensor pre_bias, std::string norm, double eps) {
  refuse_modes("block_norm", x, plain(res_), plain(gate_), plain(post_scale),
               plain(post_bias), plain(pre_scale), plain(pre_bias));
  REFUSE_UNLESS(x.dim() >= 1 && dtype_ok(x),
                "block_norm: x must be [..., D] in float32, bfloat16 or "
                "float16, got ", x.scalar_type(), " ", x.sizes());
  const int64_t D = x.size(-1);
  REFUSE_UNLESS(D > 0 && D <= 16384,
                "block_norm: the width must be 1..16384, got ", D);
  Tensor res = plain(res_);
  if (res.defined())
    REFUSE_UNLESS(res.sizes() == x.sizes() &&
                      res.scalar_type() == x.scalar_type() &&
                      res.device() == x.device(),
                  "block_norm: res must have x's shape, dtype and device");
  REFUSE_UNLESS(norm == "layer" || norm == "rms",
                "block_norm: norm must be layer or rms, got '", norm, "'");
  REFUSE_UNLESS(gate_kind == "scale" || gate_kind == "highway",
                "block_norm: gate_kind must be scale or highway, got '",
                gate_kind, "'");
  REFUSE_UNLESS(res.defined() || gate_kind != "highway",
                "block_norm: a highway needs res");
  Tensor gate = plain(gate_);
  bool channel_gate = false;
  if (gate.defined()) {
    channel_gate = gate.dim() == 1 && gate.size(0) == D && x.dim() > 1;
    REFUSE_UNLESS(channel_gate || (gate.sizes() == x.sizes() &&
                                   gate.scalar_type() == x.scalar_type() &&
                                   gate.device() == x.device()),
                  "block_norm: gate must be [D] or of x's shape and dtype, "
                  "got ", gate.scalar_type(), " ", gate.sizes());
  }
  REFUSE_UNLESS(post_scale.has_value() || !post_bias.has_value(),
                "block_norm: post_bias needs post_scale");
  REFUSE_UNLESS(pre_scale.has_value() || !pre_bias.has_value(),
                "block_norm: pre_bias needs pre_scale");
  Tensor vec[4] = {plain(post_scale), plain(post_bias), plain(pre_scale),
                   plain(pre_bias)};
  c10::optional<c10::ScalarType> pdt;
  auto check_vec = [&](Tensor& v) {
    if (!v.defined()) return;
    REFUSE_UNLESS(v.dim() == 1 && v.size(0) == D && v.device() == x.device(),
                  "block_norm: parameters must be [", D, "] on x's device");
    const auto s = v.scalar_type();
    REFUSE_UNLESS((s == x.scalar_type() || s == torch::kFloat32) &&
                      (!pdt.has_value() || *pdt == s),
                  "block_norm: parameters must share one dtype, x's or "
                  "float32");
    pdt = s;
    v = v.contiguous();
  };
  for (auto& v : vec) check_vec(v);
  if (channel_gate)
    check_vec(gate);
  else if (gate.defined())
    gate = gate.contiguous();
  x = x.contiguous();
  if (res.defined()) res = res.contiguous();
  const bool highway = gate_kind == "highway", rms = norm == "rms";
  bool grad = wants_grad(x) || wants_grad(res) || wants_grad(gate);
  for (auto& v : vec) grad = grad || wants_grad(v);
  if (grad && c10::GradMode::is_enabled()) {
    auto out = JoinFn::apply(x, opt(res), opt(gate), opt(vec[0]), opt(vec[1]),
                             opt(vec[2]), opt(vec[3]), channel_gate, highway,
                             alpha, rms, eps);
    return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
  }
  const at::NoGradGuard no_grad;
  auto out = block_norm_fwd(x.sizes(), rows(x), rows(opt(res), false),
                            rows(opt(gate), channel_gate), highway, alpha,
                            opt(vec[0]), opt(vec[1]), opt(vec[2]), opt(vec[3]),
                            rms, eps, false);
  return {out[0], opt(out[1])};
}
