// Host side of the fused block join (kernels: block_norm.h) and the sum of
// its parameter gradients.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "block_norm.h"
#include "fresh.h"

using namespace mamd;

namespace mamd {
extern template int join_fwd_launch<bf16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template int join_fwd_launch<f16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template int join_fwd_launch<float>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template int join_bwd_launch<bf16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template int join_bwd_launch<f16_t>(const NormPlan&, unsigned,
                                            hipStream_t);
extern template int join_bwd_launch<float>(const NormPlan&, unsigned,
                                            hipStream_t);
}  // namespace mamd

namespace {

struct SumArgs {
  const float* part;
  int n, D;
  int slot[kNumSums];
  int gate;                  // kNone unless the gate is per channel
  const void* gate_p;        // parameters as in NormArgs
  const void* w1;
  void* out[kNumSums];       // dgate, dpost_scale, .._bias, dpre_scale, .._bias
};

// The blocks' partial sums, and the parameter gradients from them: 16 columns
// per block, its 64 lane groups take every 64th row and meet in LDS, always in
// the same order.
template <typename P, int NP>
__global__ __launch_bounds__(1024) void param_sum_kernel(SumArgs a) {
  __shared__ float buf[NP][64][17];
  __shared__ float total[NP][16];
  const int lane = threadIdx.x & 15, grp = threadIdx.x / 16;
  const int c = blockIdx.x * 16 + lane;
  float t[NP] = {};
  if (c < a.D) {
#pragma unroll 4
    for (int i = grp; i < a.n; i += 64) {
      const float* row = a.part + (size_t)i * NP * a.D + c;
#pragma unroll
      for (int p = 0; p < NP; ++p) t[p] += row[(size_t)p * a.D];
    }
  }
#pragma unroll
  for (int p = 0; p < NP; ++p) buf[p][grp][lane] = t[p];
  __syncthreads();
  if (grp < NP) {  // group p adds up the p-th sum
    float v[16] = {};  // 16 runs of 4, then pairs: fewer roundings a term
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i % 16] += buf[grp][i][lane];
#pragma unroll
    for (int k = 8; k > 0; k /= 2)
#pragma unroll
      for (int i = 0; i < k; ++i) v[i] += v[i + k];
    total[grp][lane] = v[0];
  }
  __syncthreads();
  if (grp != 0 || c >= a.D) return;
  float sum[kNumSums];
#pragma unroll
  for (int p = 0; p < kNumSums; ++p)
    sum[p] = a.slot[p] >= 0 ? total[a.slot[p]][lane] : 0.f;
  const float s1 = sum[kS1], s0 = sum[kS0];
  const float w1 = a.w1 ? (float)((const P*)a.w1)[c] : 1.f;
  float b = 1.f, dg = 0.f;
  if (a.gate != kNone) {
    const float g = (float)((const P*)a.gate_p)[c];
    if (a.gate == kHighCh) {
      float k1;
      sigmoid2<float>(g, b, k1);
      dg = b * k1 * sum[kS2];
    } else {
      b = g;
      dg = a.slot[kS2] >= 0 ? sum[kS2] : w1 * s1;
    }
  }
  const float o[kNumSums] = {dg, b * s1, b * s0, sum[kP1], sum[kP0]};
#pragma unroll
  for (int p = 0; p < kNumSums; ++p)
    if (a.out[p]) ((P*)a.out[p])[c] = (P)o[p];
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

NormPlan make_plan(const torch::Tensor& x,
                   const c10::optional<torch::Tensor>& res,
               const c10::optional<torch::Tensor>& gate, bool highway,
               double alpha, const c10::optional<torch::Tensor>& post_scale,
               const c10::optional<torch::Tensor>& post_bias,
               const c10::optional<torch::Tensor>& pre_scale,
               const c10::optional<torch::Tensor>& pre_bias, bool rms,
               double eps, bool bwd) {
  NormPlan pl;
  NormArgs& a = pl.a;
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(),
              "block_norm: x must be dense [R, D] on a GPU");
  if (res.has_value()) check_like(*res, x, "res");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) <= 16384,
              "block_norm: the width must be 1..16384, got ", x.size(1));
  a.rows = x.size(0), a.D = x.size(1);
  a.x = x.data_ptr();
  a.res = res.has_value() ? res->data_ptr() : nullptr;
  bool seen = false;
  if (gate.has_value()) {
    if (gate->dim() == 1) {
      pl.gate = highway ? kHighCh : kScaleCh;
      a.gate = param_ptr(gate, x, a.param32, seen, "gate");
    } else {
      pl.gate = highway ? kHighTok : kScaleTok;
      check_like(*gate, x, "gate");
      a.gate = gate->data_ptr();
    }
  }
  a.post_scale = param_ptr(post_scale, x, a.param32, seen, "post_scale");
  a.post_bias = param_ptr(post_bias, x, a.param32, seen, "post_bias");
  a.pre_scale = param_ptr(pre_scale, x, a.param32, seen, "pre_scale");
  a.pre_bias = param_ptr(pre_bias, x, a.param32, seen, "pre_bias");
  a.rms = rms;
  a.alpha = (float)alpha;
  a.eps = (float)eps;
  // A row's lanes: part of a wave up to 256 columns, a wave of 8 elements a
  // lane up to 512, then a block of 8 elements a lane, 16 from 4097 columns
  // on. The forward pass takes one wave up to 1024 columns of 16 bits (16
  // elements a lane, no barriers: 110 us at 65536 x 1024 where two waves take
  // 130); the backward pass would need 291 registers for that.
  const int vec = x.element_size() == 2 ? 8 : 4;
  if (a.D < vec) {
    pl.ept = 1;
    pl.place = kPartWave;
  } else if (a.D <= 256) {
    pl.place = kPartWave;
  } else if (a.D <= 512) {
    pl.place = kWave;
  } else if (a.D <= 1024 && vec == 8 && !bwd) {
    pl.ept = 16;
    pl.place = kWave;
  } else {
    pl.ept = a.D <= 4096 ? 8 : 16;
    pl.place = kBlock;
  }
  a.tpr = 1;
  while (a.tpr * pl.ept < a.D) a.tpr *= 2;
  if (pl.place == kWave) a.tpr = WAVE;
  // Two rows a block where the backward pass takes two waves each: half the
  // partial sums to write and to add up (65536 x 1024 bf16
  // with four sums: 173 us for 192).
  if (bwd && pl.place == kBlock && a.tpr == 128) pl.place = kPair;
  pl.threads = pl.place == kBlock ? a.tpr : 256;
  pl.rpb = pl.threads / a.tpr;
  return pl;
}

int dispatch(bool bwd, const torch::Tensor& x, const NormPlan& pl,
             unsigned grid) {
  auto stream = at::cuda::getCurrentHIPStream();
  int n = 0;
  if (x.scalar_type() == torch::kBFloat16)
    n = bwd ? join_bwd_launch<bf16_t>(pl, grid, stream)
            : join_fwd_launch<bf16_t>(pl, grid, stream);
  else if (x.scalar_type() == torch::kHalf)
    n = bwd ? join_bwd_launch<f16_t>(pl, grid, stream)
            : join_fwd_launch<f16_t>(pl, grid, stream);
  else if (x.scalar_type() == torch::kFloat32)
    n = bwd ? join_bwd_launch<float>(pl, grid, stream)
            : join_fwd_launch<float>(pl, grid, stream);
  else
    TORCH_CHECK(false, "block_norm: unsupported dtype");
  TORCH_CHECK(n > 0, "block_norm: no kernel for this plan");
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return n;
}

// The blocks that the GPU holds at once, which walk over the rows: more would
// run as a second, partly filled round (125 us for 110 at 65536 x 1024 bf16
// forward without a gate), and the backward pass writes partial sums for each.
unsigned grid_of(bool bwd, const torch::Tensor& x, const NormPlan& pl,
                 int min_rows) {
  const long all = (pl.a.rows + pl.rpb - 1) / pl.rpb;
  const long cus = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  if (all <= cus) return (unsigned)all;
  const long few = std::max((all + min_rows - 1) / min_rows, cus);
  return (unsigned)std::min(few, cus * dispatch(bwd, x, pl, 0));
}

}  // namespace

// returns (s, h, stat): h is undefined without pre_scale, stat without
// want_stat; s and h have `sizes`, x's before its rows were laid out
std::vector<torch::Tensor> block_norm_fwd(
    at::IntArrayRef sizes, torch::Tensor x, c10::optional<torch::Tensor> res,
    c10::optional<torch::Tensor> gate,
    bool highway, double alpha, c10::optional<torch::Tensor> post_scale,
    c10::optional<torch::Tensor> post_bias,
    c10::optional<torch::Tensor> pre_scale,
    c10::optional<torch::Tensor> pre_bias, bool rms, double eps,
    bool want_stat) {
  NormPlan pl = make_plan(x, res, gate, highway, alpha, post_scale, post_bias,
                      pre_scale, pre_bias, rms, eps, false);
  NormArgs& a = pl.a;
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK(c10::multiply_integers(sizes) == x.numel(),
              "block_norm: sizes are not x's");
  auto s = fresh(sizes, x.scalar_type(), x);
  torch::Tensor h, stat;
  if (a.pre_scale) h = fresh_like(s), a.h = h.data_ptr();
  if (want_stat) {
    stat = fresh({4, a.rows}, torch::kFloat32, x);
    a.stat = stat.data_ptr<float>();
  }
  if (a.rows == 0) return {s, h, stat};
  a.s = s.data_ptr();
  dispatch(false, x, pl, grid_of(false, x, pl, 1));
  return {s, h, stat};
}

// returns (dx, dres, dgate, dpost_scale, dpost_bias, dpre_scale, dpre_bias);
// those that `want` (same order) does not ask for are undefined
std::vector<torch::Tensor> block_norm_bwd(
    torch::Tensor x, c10::optional<torch::Tensor> res,
    c10::optional<torch::Tensor> gate,
    bool highway, double alpha, c10::optional<torch::Tensor> post_scale,
    c10::optional<torch::Tensor> post_bias,
    c10::optional<torch::Tensor> pre_scale,
    c10::optional<torch::Tensor> pre_bias, bool rms, double eps,
    torch::Tensor stat, c10::optional<torch::Tensor> dsum,
    c10::optional<torch::Tensor> dh, std::vector<bool> want) {
  NormPlan pl = make_plan(x, res, gate, highway, alpha, post_scale, post_bias,
                      pre_scale, pre_bias, rms, eps, true);
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
  std::vector<torch::Tensor> out(7);
  if (want[0]) out[0] = fresh_like(x), a.dx = out[0].data_ptr();
  if (want[1] && a.res) out[1] = fresh_like(x), a.dres = out[1].data_ptr();
  const bool channel = is_channel(pl.gate);
  if (want[2] && is_token(pl.gate))
    out[2] = fresh_like(x), a.dgate = out[2].data_ptr();
  SumArgs sm{};
  const auto pdt = a.param32 ? torch::kFloat32 : x.scalar_type();
  auto vec = [&](int at, bool there) {
    if (!want[at] || !there) return false;
    out[at] = fresh({a.D}, pdt, x);
    sm.out[at - 2] = out[at].data_ptr();
    return true;
  };
  const bool dg = vec(2, channel), dw1 = vec(3, a.post_scale),
             db1 = vec(4, a.post_bias), dw2 = vec(5, a.pre_scale),
             db2 = vec(6, a.pre_bias);
  const bool terms = pl.gate == kHighCh || a.post_bias;
  const bool use[kNumSums] = {dw1 || (dg && !terms), db1, dg && terms, dw2,
                              db2};
  for (int p = 0; p < kNumSums; ++p)
    sm.slot[p] = a.slot[p] = use[p] ? a.n_part++ : -1;
  if (a.rows == 0) {
    for (auto& t : out)
      if (t.defined()) t.zero_();
    return out;
  }
  // 4 turns at least for each block: one turn's partial sums are as many
  // bytes as most of what it reads
  const unsigned grid = grid_of(true, x, pl, a.n_part ? 4 : 1);
  torch::Tensor part;
  if (a.n_part) {
    part = fresh({(long)grid, a.n_part, a.D}, torch::kFloat32, x);
    a.part = part.data_ptr<float>();
  }
  dispatch(true, x, pl, grid);
  if (a.n_part) {
    sm.part = a.part;
    sm.n = grid, sm.D = a.D;
    sm.gate = channel ? pl.gate : kNone;
    sm.gate_p = a.gate, sm.w1 = a.post_scale;
    const unsigned sgrid = (unsigned)((a.D + 15) / 16);
    auto stream = at::cuda::getCurrentHIPStream();
#define SUMN(P, NP)                                                          \
  case NP:                                                                   \
    hipLaunchKernelGGL((param_sum_kernel<P, NP>), dim3(sgrid), dim3(1024),   \
                       0, stream, sm);                                       \
    break;
#define SUM(P)                                                               \
  switch (a.n_part) {                                                        \
    SUMN(P, 1) SUMN(P, 2) SUMN(P, 3) SUMN(P, 4) SUMN(P, 5)                   \
  }
    if (a.param32 || x.scalar_type() == torch::kFloat32) { SUM(float) }
    else if (x.scalar_type() == torch::kBFloat16) { SUM(bf16_t) }
    else { SUM(f16_t) }
#undef SUM
#undef SUMN
    C10_HIP_KERNEL_LAUNCH_CHECK();
  }
  return out;
}
