// Host side of the fused block join (kernels: block_norm.h) and the sum of
// its parameter gradients.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "block_norm.h"

using namespace mamd;

namespace mamd {
extern template void join_fwd_launch<bf16_t>(const NormPlan&, unsigned,
                                             hipStream_t);
extern template void join_fwd_launch<f16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template void join_fwd_launch<float>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template void join_bwd_launch<bf16_t>(const NormPlan&, unsigned,
                                             hipStream_t);
extern template void join_bwd_launch<f16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template void join_bwd_launch<float>(const NormPlan&, unsigned,
                                            hipStream_t);
}  // namespace mamd

#define NORM_DTYPES(st, FN)                                             \
  if (st == torch::kBFloat16) FN<bf16_t>(pl, grid, stream);             \
  else if (st == torch::kHalf) FN<f16_t>(pl, grid, stream);             \
  else if (st == torch::kFloat32) FN<float>(pl, grid, stream);          \
  else TORCH_CHECK(false, "block_norm: unsupported dtype");

namespace {

struct SumArgs {
  const float* part;
  int n, n_part, D;
  void* out[kNumParams];
};

// the blocks' partial sums: 64 columns per block, its 16 waves take every
// 16th row and meet in LDS, always in the same order
template <typename P>
__global__ __launch_bounds__(1024) void param_sum_kernel(SumArgs a) {
  __shared__ float buf[16][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x / 64;
  const int cols = (a.D + 63) / 64;
  const int p = blockIdx.x / cols, c = (blockIdx.x % cols) * 64 + lane;
  float t = 0.f;
  if (c < a.D) {
#pragma unroll 4
    for (int i = wid; i < a.n; i += 16)
      t += a.part[((size_t)i * a.n_part + p) * a.D + c];
  }
  buf[wid][lane] = t;
  __syncthreads();
  if (wid == 0 && c < a.D) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += buf[i][lane];
    ((P*)a.out[p])[c] = (P)t;
  }
}

const void* param_ptr(const c10::optional<torch::Tensor>& p,
                      const torch::Tensor& x, int& param32, bool& seen,
                      const char* what) {
  if (!p.has_value()) return nullptr;
  TORCH_CHECK(p->device() == x.device() && p->is_contiguous() &&
                  p->dim() == 1 && p->size(0) == x.size(-1),
              "block_norm: ", what, " must be dense [D] on x's device");
  const bool f32 = p->scalar_type() == torch::kFloat32;
  TORCH_CHECK(f32 || p->scalar_type() == x.scalar_type(), "block_norm: ", what,
              " must be float32 or of x's dtype");
  TORCH_CHECK(!seen || param32 == (int)f32,
              "block_norm: parameters must share a dtype");
  param32 = f32;
  seen = true;
  return p->data_ptr();
}

void check_like(const torch::Tensor& t, const torch::Tensor& x,
                const char* what) {
  TORCH_CHECK(t.device() == x.device() && t.sizes() == x.sizes() &&
                  t.scalar_type() == x.scalar_type() && t.is_contiguous(),
              "block_norm: ", what, " must be dense and like x");
}

NormPlan make_plan(const torch::Tensor& x, const torch::Tensor& res,
               const c10::optional<torch::Tensor>& gate, bool highway,
               double alpha, const c10::optional<torch::Tensor>& post_scale,
               const c10::optional<torch::Tensor>& post_bias,
               const c10::optional<torch::Tensor>& pre_scale,
               const c10::optional<torch::Tensor>& pre_bias, bool rms,
               double eps) {
  NormPlan pl;
  NormArgs& a = pl.a;
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(),
              "block_norm: x must be dense [R, D] on a GPU");
  check_like(res, x, "res");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) <= 16384,
              "block_norm: the width must be 1..16384, got ", x.size(1));
  a.rows = x.size(0), a.D = x.size(1);
  a.x = x.data_ptr();
  a.res = res.data_ptr();
  bool seen = false;
  if (gate.has_value()) {
    if (gate->dim() == 1) {
      pl.gate_mode = kGateChannel;
      a.gate = param_ptr(gate, x, a.param32, seen, "gate");
    } else {
      pl.gate_mode = kGateToken;
      check_like(*gate, x, "gate");
      a.gate = gate->data_ptr();
    }
  }
  a.post_scale = param_ptr(post_scale, x, a.param32, seen, "post_scale");
  a.post_bias = param_ptr(post_bias, x, a.param32, seen, "post_bias");
  a.pre_scale = param_ptr(pre_scale, x, a.param32, seen, "pre_scale");
  a.pre_bias = param_ptr(pre_bias, x, a.param32, seen, "pre_bias");
  a.highway = highway;
  a.rms = rms;
  a.alpha = (float)alpha;
  a.eps = (float)eps;
  // a row's lanes: 8 elements each up to 4096, 16 above
  pl.ept = a.D <= 4096 ? 8 : 16;
  a.tpr = 1;
  while (a.tpr * pl.ept < a.D) a.tpr *= 2;
  pl.threads = a.tpr > WAVE ? a.tpr : 256;
  pl.rpb = pl.threads / a.tpr;
  return pl;
}

}  // namespace

// returns (s, h, stat): h is empty without pre_scale, stat without want_stat
std::vector<torch::Tensor> block_norm_fwd(
    torch::Tensor x, torch::Tensor res, c10::optional<torch::Tensor> gate,
    bool highway, double alpha, c10::optional<torch::Tensor> post_scale,
    c10::optional<torch::Tensor> post_bias,
    c10::optional<torch::Tensor> pre_scale,
    c10::optional<torch::Tensor> pre_bias, bool rms, double eps,
    bool want_stat) {
  NormPlan pl = make_plan(x, res, gate, highway, alpha, post_scale, post_bias,
                      pre_scale, pre_bias, rms, eps);
  NormArgs& a = pl.a;
  const c10::DeviceGuard guard(x.device());
  auto s = torch::empty_like(x);
  auto h = a.pre_scale ? torch::empty_like(x) : torch::empty({0}, x.options());
  auto stat = torch::empty({want_stat ? 4 : 0, (long)a.rows},
                           x.options().dtype(torch::kFloat32));
  if (a.rows == 0) return {s, h, stat};
  a.s = s.data_ptr();
  a.h = h.data_ptr();
  a.stat = want_stat ? stat.data_ptr<float>() : nullptr;
  const long blocks = (a.rows + pl.rpb - 1) / pl.rpb;
  const unsigned grid = (unsigned)std::min<long>(blocks, 1L << 20);
  auto stream = at::cuda::getCurrentHIPStream();
  NORM_DTYPES(x.scalar_type(), join_fwd_launch)
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {s, h, stat};
}

// returns (dx, dres, dgate, dpost_scale, dpost_bias, dpre_scale, dpre_bias);
// those that `want` (same order) does not ask for are empty
std::vector<torch::Tensor> block_norm_bwd(
    torch::Tensor x, torch::Tensor res, c10::optional<torch::Tensor> gate,
    bool highway, double alpha, c10::optional<torch::Tensor> post_scale,
    c10::optional<torch::Tensor> post_bias,
    c10::optional<torch::Tensor> pre_scale,
    c10::optional<torch::Tensor> pre_bias, bool rms, double eps,
    torch::Tensor stat, c10::optional<torch::Tensor> dsum,
    c10::optional<torch::Tensor> dh, std::vector<bool> want) {
  NormPlan pl = make_plan(x, res, gate, highway, alpha, post_scale, post_bias,
                      pre_scale, pre_bias, rms, eps);
  NormArgs& a = pl.a;
  TORCH_CHECK(want.size() == 7, "block_norm_bwd: want must have 7 entries");
  TORCH_CHECK(stat.device() == x.device() &&
                  stat.scalar_type() == torch::kFloat32 &&
                  stat.is_contiguous() && stat.numel() == 4 * a.rows,
              "block_norm_bwd: stat is not this forward pass's");
  const c10::DeviceGuard guard(x.device());
  a.stat = stat.data_ptr<float>();
  torch::Tensor dsc, dhc;
  if (dsum.has_value()) {
    dsc = dsum->contiguous();
    check_like(dsc, x, "dsum");
    a.dsum = dsc.data_ptr();
  }
  if (dh.has_value() && a.pre_scale) {
    dhc = dh->contiguous();
    check_like(dhc, x, "dh");
    a.dh = dhc.data_ptr();
  }
  auto none = torch::empty({0}, x.options());
  std::vector<torch::Tensor> out(7, none);
  if (want[0]) out[0] = torch::empty_like(x), a.dx = out[0].data_ptr();
  if (want[1]) out[1] = torch::empty_like(x), a.dres = out[1].data_ptr();
  if (want[2] && pl.gate_mode == kGateToken)
    out[2] = torch::empty_like(x), a.dgate = out[2].data_ptr();
  SumArgs sm{};
  auto popt = x.options().dtype(a.param32 ? torch::kFloat32 : x.scalar_type());
  auto vec = [&](int param, int at, bool there) {
    a.slot[param] = -1;
    if (!want[at] || !there) return;
    out[at] = torch::empty({a.D}, popt);
    sm.out[a.n_part] = out[at].data_ptr();
    a.slot[param] = a.n_part++;
  };
  vec(kGate, 2, pl.gate_mode == kGateChannel);
  vec(kPostScale, 3, a.post_scale);
  vec(kPostBias, 4, a.post_bias);
  vec(kPreScale, 5, a.pre_scale);
  vec(kPreBias, 6, a.pre_bias);
  if (a.rows == 0) {
    for (auto& t : out) t.zero_();
    return out;
  }
  const long blocks = (a.rows + pl.rpb - 1) / pl.rpb;
  const unsigned grid =
      (unsigned)std::min<long>(blocks, a.n_part ? 1024 : 1L << 20);
  torch::Tensor part;
  if (a.n_part) {
    part = torch::empty({(long)grid, a.n_part, a.D},
                        x.options().dtype(torch::kFloat32));
    a.part = part.data_ptr<float>();
  }
  auto stream = at::cuda::getCurrentHIPStream();
  NORM_DTYPES(x.scalar_type(), join_bwd_launch)
  C10_HIP_KERNEL_LAUNCH_CHECK();
  if (a.n_part) {
    sm.part = a.part;
    sm.n = grid, sm.n_part = a.n_part, sm.D = a.D;
    const unsigned sgrid = (unsigned)(((a.D + 63) / 64) * a.n_part);
#define SUM(P)                                                               \
  hipLaunchKernelGGL((param_sum_kernel<P>), dim3(sgrid), dim3(1024), 0,      \
                     stream, sm)
    if (a.param32 || x.scalar_type() == torch::kFloat32) { SUM(float); }
    else if (x.scalar_type() == torch::kBFloat16) { SUM(bf16_t); }
    else { SUM(f16_t); }
#undef SUM
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return out;
}
