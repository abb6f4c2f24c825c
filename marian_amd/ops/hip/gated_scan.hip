// Gated linear recurrence over sequences and its gradient, for CDNA4 (gfx950).
// ref semantics: src/rnn/cells.h SSRU, whose highway(cell, x, f) this is.
//
//   f_t = sigmoid(g_t)    c_t = f_t c_{t-1} + (1 - f_t) x_t    y_t = act(c_t)
//
// A run of steps maps the state it starts from to the one it ends in by
// c -> A c + H with A the product of its f; two runs join to
// (A' A, A' H + H'). So a thread folds a few steps, a block joins its threads
// over the time axis in LDS, and every thread then replays its steps from the
// state it really starts from. All of it is held in 32 bits.
//
// Backward: lam_t = dy_t act'(c_t) + mu_{t+1}, mu_t = f_t lam_t (mu behind the
// last step is the last state's gradient) is the same recurrence from the
// other end; dx_t = (1 - f_t) lam_t, dg_t = f_t (1 - f_t)(c_{t-1} - x_t) lam_t.
// The states are folded again from x and g, which have to be read anyway,
// starting at the 32-bit states that the forward pass kept at each tile's
// start: no full-size state tensor is written or read.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "common.h"
#include "vec.h"

using namespace mamd;

namespace {

struct ScanArgs {
  const void* x;
  const void* g;
  long xb, xt, gb, gt;      // strides of batch and time, in elements
  const float* state;       // [B,D] or null (zeros)
  const int* lens;          // [B] or null (T)
  float* bnd;               // [B,nt,D] state at each tile's start, or null
  int B, T, D;
  int nt;                   // tiles of kTile steps
  int reverse, relu;
  // forward
  void* y;                  // [B,T,D] contiguous
  float* last;              // [B,D]
  // backward
  const void* dy;           // [B,T,D] contiguous or null
  const float* dlast;       // [B,D] or null
  void* dx;
  void* dg;
  long dxb, dxt, dgb, dgt;
  float* dstate;            // [B,D] or null
};

// a tile's steps; the forward and the backward pass agree on it, since one
// keeps the states that the other starts from
constexpr int kTile = 64;

__device__ __forceinline__ int valid_len(const ScanArgs& a, int b) {
  return a.lens ? min(max(a.lens[b], 0), a.T) : a.T;
}

// step s of the recurrence sits at this position of the time axis
__device__ __forceinline__ int time_of(const ScanArgs& a, int s, int len) {
  return a.reverse ? len - 1 - s : s;
}

// a NaN state stays visible, which fmaxf would turn into 0
__device__ __forceinline__ float activate(float c, int relu) {
  return relu && c < 0.f ? 0.f : c;
}

// Block: LC lanes of VEC channels by SUB groups of STEPS steps. A lane whose
// channels would pass the row's end moves back to the last VEC channels: it
// computes what its neighbours compute and writes the same values there, so
// every access is whole and in bounds for any D >= VEC. Steps behind the
// sequence read position 0 and are masked.
template <int VEC, int LC>
__device__ __forceinline__ int lane_channel(const ScanArgs& a, int ctile,
                                            int lc, bool& owns) {
  const int ch = ctile * (LC * VEC) + lc * VEC;
  owns = ch < a.D;
  return min(ch, a.D - VEC);
}

template <typename T, int VEC, int LC, int SUB>
__global__ __launch_bounds__(LC* SUB) void scan_fwd_kernel(ScanArgs a,
                                                           int ctiles) {
  constexpr int STEPS = kTile / SUB;
  __shared__ float sA[SUB][LC * VEC], sH[SUB][LC * VEC];
  const int lc = threadIdx.x % LC, sub = threadIdx.x / LC;
  const int b = blockIdx.x / ctiles;
  bool owns;
  const int ch = lane_channel<VEC, LC>(a, blockIdx.x % ctiles, lc, owns);
  const int len = valid_len(a, b);
  const T* x = (const T*)a.x + (size_t)b * a.xb + ch;
  const T* g = (const T*)a.g + (size_t)b * a.gb + ch;
  T* y = (T*)a.y + (size_t)b * a.T * a.D + ch;
  const size_t vec0 = (size_t)b * a.D + ch;  // this lane in a [B,D] array

  float c[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) c[v] = a.state ? a.state[vec0 + v] : 0.f;

  for (int tile = 0; tile < a.nt; ++tile) {
    const int s0 = tile * kTile + sub * STEPS;
    if (a.bnd && sub == 0 && owns)
      store_vec<float, VEC>(a.bnd + ((size_t)b * a.nt + tile) * a.D + ch, c);
    vec_t<T, VEC> xr[STEPS], gr[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int s = s0 + j;
      const int t = s < len ? time_of(a, s, len) : 0;
      xr[j] = load_vec<T, VEC>(x + (size_t)t * a.xt);
      gr[j] = load_vec<T, VEC>(g + (size_t)t * a.gt);
    }
    float f[STEPS][VEC], h[STEPS][VEC];
    float A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const bool on = s0 + j < len;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float ff, om;
        sigmoid2<T>((float)gr[j][v], ff, om);
        f[j][v] = on ? ff : 1.f;  // a padded step holds the state
        h[j][v] = on ? om * (float)xr[j][v] : 0.f;
        A[v] *= f[j][v];
        H[v] = f[j][v] * H[v] + h[j][v];
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      sA[sub][lc * VEC + v] = A[v];
      sH[sub][lc * VEC + v] = H[v];
    }
    __syncthreads();
    float cur[VEC];
#pragma unroll
    for (int k = 0; k < SUB; ++k) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (k == sub) cur[v] = c[v];
        c[v] = sA[k][lc * VEC + v] * c[v] + sH[k][lc * VEC + v];
      }
    }
    __syncthreads();
    if (owns) {
#pragma unroll
      for (int j = 0; j < STEPS; ++j) {
        const int s = s0 + j;
        float o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          cur[v] = f[j][v] * cur[v] + h[j][v];
          o[v] = s < len ? activate(cur[v], a.relu) : 0.f;
        }
        if (s < a.T)
          store_vec<T, VEC>(
              y + (size_t)(s < len ? time_of(a, s, len) : s) * a.D, o);
      }
    }
  }
  if (sub == 0 && owns) store_vec<float, VEC>(a.last + vec0, c);
}

template <typename T, int VEC, int LC, int SUB>
__global__ __launch_bounds__(LC* SUB) void scan_bwd_kernel(ScanArgs a,
                                                           int ctiles) {
  constexpr int STEPS = kTile / SUB;
  __shared__ float sA[SUB][LC * VEC], sH[SUB][LC * VEC], sM[SUB][LC * VEC];
  const int lc = threadIdx.x % LC, sub = threadIdx.x / LC;
  const int b = blockIdx.x / ctiles;
  bool owns;
  const int ch = lane_channel<VEC, LC>(a, blockIdx.x % ctiles, lc, owns);
  const int len = valid_len(a, b);
  const T* x = (const T*)a.x + (size_t)b * a.xb + ch;
  const T* g = (const T*)a.g + (size_t)b * a.gb + ch;
  const T* dy = a.dy ? (const T*)a.dy + (size_t)b * a.T * a.D + ch : nullptr;
  T* dx = (T*)a.dx + (size_t)b * a.dxb + ch;
  T* dg = (T*)a.dg + (size_t)b * a.dgb + ch;
  const size_t vec0 = (size_t)b * a.D + ch;

  float mu[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) mu[v] = a.dlast ? a.dlast[vec0 + v] : 0.f;

  for (int tile = a.nt - 1; tile >= 0; --tile) {
    const int s0 = tile * kTile + sub * STEPS;
    vec_t<T, VEC> xr[STEPS], gr[STEPS], dr[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const int s = s0 + j;
      const int t = s < len ? time_of(a, s, len) : 0;
      xr[j] = load_vec<T, VEC>(x + (size_t)t * a.xt);
      gr[j] = load_vec<T, VEC>(g + (size_t)t * a.gt);
      dr[j] = {};
      if (dy) dr[j] = load_vec<T, VEC>(dy + (size_t)t * a.D);
    }
    // the state at this tile's start
    const float* cp = a.bnd ? a.bnd + ((size_t)b * a.nt + tile) * a.D + ch
                            : (a.state ? a.state + vec0 : nullptr);
    float A[VEC], H[VEC], c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = 1.f, H[v] = 0.f;
      c[v] = cp ? cp[v] : 0.f;
    }
    float f[STEPS][VEC], om[STEPS][VEC], w[STEPS][VEC], d[STEPS][VEC];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) {
      const bool on = s0 + j < len;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float ff, oo;
        sigmoid2<T>((float)gr[j][v], ff, oo);
        f[j][v] = on ? ff : 1.f;
        om[j][v] = on ? oo : 0.f;
        w[j][v] = on ? (float)xr[j][v] : 0.f;
        d[j][v] = on ? (float)dr[j][v] : 0.f;
        A[v] *= f[j][v];
        H[v] = f[j][v] * H[v] + om[j][v] * w[j][v];
      }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      sA[sub][lc * VEC + v] = A[v];
      sH[sub][lc * VEC + v] = H[v];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SUB - 1; ++k)
#pragma unroll
      for (int v = 0; v < VEC; ++v)
        if (k < sub) c[v] = sA[k][lc * VEC + v] * c[v] + sH[k][lc * VEC + v];
    // w becomes c_{t-1} - x_t, d is cut where relu was off
#pragma unroll
    for (int j = 0; j < STEPS; ++j)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const float xv = w[j][v];
        w[j][v] = c[v] - xv;
        c[v] = f[j][v] * c[v] + om[j][v] * xv;
        if (a.relu && c[v] <= 0.f) d[j][v] = 0.f;
      }
    // this thread's steps from the far end, with nothing coming in
    float M[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) M[v] = 0.f;
#pragma unroll
    for (int j = STEPS - 1; j >= 0; --j)
#pragma unroll
      for (int v = 0; v < VEC; ++v) M[v] = f[j][v] * (d[j][v] + M[v]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) sM[sub][lc * VEC + v] = M[v];
    __syncthreads();
    float cur[VEC];
#pragma unroll
    for (int k = SUB - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (k == sub) cur[v] = mu[v];
        mu[v] = sA[k][lc * VEC + v] * mu[v] + sM[k][lc * VEC + v];
      }
    __syncthreads();
    if (owns) {
#pragma unroll
      for (int j = STEPS - 1; j >= 0; --j) {
        const int s = s0 + j;
        float ox[VEC], og[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float lam = d[j][v] + cur[v];
          cur[v] = f[j][v] * lam;
          ox[v] = s < len ? om[j][v] * lam : 0.f;
          og[v] = s < len ? cur[v] * om[j][v] * w[j][v] : 0.f;
        }
        if (s < a.T) {
          const int t = s < len ? time_of(a, s, len) : s;
          store_vec<T, VEC>(dx + (size_t)t * a.dxt, ox);
          store_vec<T, VEC>(dg + (size_t)t * a.dgt, og);
        }
      }
    }
  }
  if (a.dstate && sub == 0 && owns)
    store_vec<float, VEC>(a.dstate + vec0, mu);
}

// one token for each row: the recurrence at T = 1, on a pool of states.
// Here the last vector of a row goes element by element: in place, a state
// must be read and written by one thread only.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void step_kernel(
    const T* __restrict__ x, const T* __restrict__ g, long xs, long gs,
    const float* state, float* state_out, T* __restrict__ y, long n_vec,
    int vpr, int D, int relu) {
  const long i = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_vec) return;
  const long row = i / vpr;
  const int ch = (int)(i - row * vpr) * VEC;
  const T* xp = x + row * xs + ch;
  const T* gp = g + row * gs + ch;
  const size_t at = (size_t)row * D + ch;
  if (ch + VEC <= D) {
    const vec_t<T, VEC> xv = load_vec<T, VEC>(xp), gv = load_vec<T, VEC>(gp);
    const vec_t<float, VEC> cv = load_vec<float, VEC>(state + at);
    float c[VEC], o[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      float f, om;
      sigmoid2<T>((float)gv[v], f, om);
      c[v] = f * cv[v] + om * (float)xv[v];
      o[v] = activate(c[v], relu);
    }
    store_vec<float, VEC>(state_out + at, c);
    store_vec<T, VEC>(y + at, o);
  } else {
    for (int v = 0; ch + v < D; ++v) {
      float f, om;
      sigmoid2<T>((float)gp[v], f, om);
      const float c = f * state[at + v] + om * (float)xp[v];
      state_out[at + v] = c;
      y[at + v] = (T)activate(c, relu);
    }
  }
}

int act_code(const std::string& act) {
  TORCH_CHECK(act == "none" || act == "relu",
              "gated_scan: act must be none or relu, got ", act);
  return act == "relu";
}

void check_rows(const torch::Tensor& x, const torch::Tensor& g,
                const char* what) {
  TORCH_CHECK(x.is_cuda() && g.device() == x.device(), what,
              ": x and gate must be on one GPU");
  TORCH_CHECK(g.scalar_type() == x.scalar_type(), what,
              ": x and gate must share a dtype");
  TORCH_CHECK(g.sizes() == x.sizes(), what,
              ": x and gate must have the same shape");
  TORCH_CHECK(x.size(-1) > 0, what, ": the width must be positive");
  TORCH_CHECK(x.size(-1) == 1 || (x.stride(-1) == 1 && g.stride(-1) == 1),
              what, ": the last dimension must be dense");
}

const float* state_ptr(const c10::optional<torch::Tensor>& s,
                       const torch::Tensor& x, const char* what) {
  if (!s.has_value()) return nullptr;
  TORCH_CHECK(s->device() == x.device() &&
                  s->scalar_type() == torch::kFloat32 && s->is_contiguous() &&
                  s->dim() == 2 && s->size(0) == x.size(0) &&
                  s->size(1) == x.size(-1),
              "gated_scan: ", what, " must be dense float32 [B, D]");
  return s->data_ptr<float>();
}

const int* lens_ptr(const c10::optional<torch::Tensor>& l,
                    const torch::Tensor& x) {
  if (!l.has_value()) return nullptr;
  TORCH_CHECK(l->device() == x.device() && l->scalar_type() == torch::kInt32 &&
                  l->is_contiguous() && l->dim() == 1 &&
                  l->size(0) == x.size(0),
              "gated_scan: lens must be dense int32 [B]");
  return l->data_ptr<int>();
}

ScanArgs base_args(const torch::Tensor& x, const torch::Tensor& g,
                   const c10::optional<torch::Tensor>& state,
                   const c10::optional<torch::Tensor>& lens, bool reverse,
                   const std::string& act) {
  check_rows(x, g, "gated_scan");
  TORCH_CHECK(x.dim() == 3, "gated_scan: x must be [B, T, D]");
  TORCH_CHECK(x.size(0) < (1 << 30) && x.size(1) < (1 << 30) &&
                  x.size(2) < (1 << 30),
              "gated_scan: sizes must stay below 2^30");
  ScanArgs a{};
  a.x = x.data_ptr();
  a.g = g.data_ptr();
  a.xb = x.stride(0), a.xt = x.stride(1);
  a.gb = g.stride(0), a.gt = g.stride(1);
  a.state = state_ptr(state, x, "state");
  a.lens = lens_ptr(lens, x);
  a.B = x.size(0), a.T = x.size(1), a.D = x.size(2);
  a.nt = (a.T + kTile - 1) / kTile;
  a.reverse = reverse;
  a.relu = act_code(act);
  return a;
}

#define SCAN_DTYPES(st, FN)                                         \
  if (st == torch::kBFloat16) { FN(bf16_t); }                       \
  else if (st == torch::kHalf) { FN(f16_t); }                       \
  else if (st == torch::kFloat32) { FN(float); }                    \
  else TORCH_CHECK(false, "gated_scan: unsupported dtype");

int grid_of(const ScanArgs& a, int ctiles) {
  const long n = (long)a.B * ctiles;
  TORCH_CHECK(n < (1L << 31), "gated_scan: too many rows");
  return (int)n;
}

}  // namespace

// returns (y, last, bnd); bnd is empty unless want_bnd and T spans tiles
std::vector<torch::Tensor> gated_scan_fwd(torch::Tensor x, torch::Tensor gate,
                                          c10::optional<torch::Tensor> state,
                                          c10::optional<torch::Tensor> lens,
                                          bool reverse, std::string act,
                                          bool want_bnd) {
  ScanArgs a = base_args(x, gate, state, lens, reverse, act);
  const c10::DeviceGuard guard(x.device());
  auto f32 = x.options().dtype(torch::kFloat32);
  auto y = torch::empty({a.B, a.T, a.D}, x.options());
  auto last = torch::empty({a.B, a.D}, f32);
  auto bnd = torch::empty({0}, f32);
  if (want_bnd && a.nt > 1) {
    bnd = torch::empty({a.B, a.nt, a.D}, f32);
    a.bnd = bnd.data_ptr<float>();
  }
  a.y = y.data_ptr();
  a.last = last.data_ptr<float>();
  if (a.B == 0) return {y, last, bnd};
  auto stream = at::cuda::getCurrentHIPStream();
#define LAUNCH(T, VEC)                                                       \
  const int ctiles = (a.D + 64 * VEC - 1) / (64 * VEC);                      \
  hipLaunchKernelGGL((scan_fwd_kernel<T, VEC, 64, 4>),                       \
                     dim3(grid_of(a, ctiles)), dim3(256), 0, stream, a,      \
                     ctiles)
#define RUN(T)                                                               \
  if (a.D >= 4) { LAUNCH(T, 4); } else { LAUNCH(T, 1); }
  SCAN_DTYPES(x.scalar_type(), RUN)
#undef RUN
#undef LAUNCH
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {y, last, bnd};
}

// writes dx and dgate (any batch and time strides); returns dstate, empty
// unless want_dstate
torch::Tensor gated_scan_bwd(torch::Tensor x, torch::Tensor gate,
                             c10::optional<torch::Tensor> state,
                             c10::optional<torch::Tensor> lens,
                             torch::Tensor bnd,
                             c10::optional<torch::Tensor> dy,
                             c10::optional<torch::Tensor> dlast, bool reverse,
                             std::string act, torch::Tensor dx,
                             torch::Tensor dgate, bool want_dstate) {
  ScanArgs a = base_args(x, gate, state, lens, reverse, act);
  const c10::DeviceGuard guard(x.device());
  check_rows(dx, dgate, "gated_scan_bwd");
  TORCH_CHECK(dx.sizes() == x.sizes() && dx.device() == x.device() &&
                  dx.scalar_type() == x.scalar_type(),
              "gated_scan_bwd: dx must be like x");
  if (a.nt > 1) {
    TORCH_CHECK(bnd.device() == x.device() &&
                    bnd.scalar_type() == torch::kFloat32 &&
                    bnd.is_contiguous() && bnd.dim() == 3 &&
                    bnd.size(0) == a.B && bnd.size(1) == a.nt &&
                    bnd.size(2) == a.D,
                "gated_scan_bwd: bnd is not this forward pass's");
    a.bnd = bnd.data_ptr<float>();
  }
  torch::Tensor dyc;
  if (dy.has_value()) {
    TORCH_CHECK(dy->sizes() == x.sizes() && dy->device() == x.device() &&
                    dy->scalar_type() == x.scalar_type(),
                "gated_scan_bwd: dy must be like y");
    dyc = dy->contiguous();
    a.dy = dyc.data_ptr();
  }
  a.dlast = state_ptr(dlast, x, "dlast");
  a.dx = dx.data_ptr();
  a.dg = dgate.data_ptr();
  a.dxb = dx.stride(0), a.dxt = dx.stride(1);
  a.dgb = dgate.stride(0), a.dgt = dgate.stride(1);
  auto f32 = x.options().dtype(torch::kFloat32);
  auto dstate = want_dstate ? torch::empty({a.B, a.D}, f32)
                            : torch::empty({0}, f32);
  if (want_dstate) a.dstate = dstate.data_ptr<float>();
  if (a.B == 0) return dstate;
  auto stream = at::cuda::getCurrentHIPStream();
#define LAUNCH(T, VEC)                                                       \
  const int ctiles = (a.D + 64 * VEC - 1) / (64 * VEC);                      \
  hipLaunchKernelGGL((scan_bwd_kernel<T, VEC, 64, 4>),                       \
                     dim3(grid_of(a, ctiles)), dim3(256), 0, stream, a,      \
                     ctiles)
#define RUN(T)                                                               \
  if (a.D >= 2) { LAUNCH(T, 2); } else { LAUNCH(T, 1); }
  SCAN_DTYPES(x.scalar_type(), RUN)
#undef RUN
#undef LAUNCH
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return dstate;
}

// one step for N rows; state_out may be state itself
torch::Tensor gated_step(torch::Tensor x, torch::Tensor gate,
                         torch::Tensor state, torch::Tensor state_out,
                         std::string act) {
  check_rows(x, gate, "gated_step");
  TORCH_CHECK(x.dim() == 2, "gated_step: x must be [N, D]");
  const int relu = act_code(act);
  const float* sp = state_ptr(state, x, "state");
  state_ptr(state_out, x, "state_out");
  const c10::DeviceGuard guard(x.device());
  const long N = x.size(0), D = x.size(1);
  TORCH_CHECK(D < (1L << 30), "gated_step: the width must stay below 2^30");
  auto y = torch::empty({N, D}, x.options());
  if (N == 0) return y;
  auto stream = at::cuda::getCurrentHIPStream();
  const int vpr = (int)((D + 3) / 4);
  const long n_vec = N * vpr;
  const long grid = (n_vec + 255) / 256;
  TORCH_CHECK(grid < (1L << 31), "gated_step: too many rows");
#define RUN(T)                                                               \
  hipLaunchKernelGGL((step_kernel<T, 4>), dim3((unsigned)grid), dim3(256),   \
                     0, stream, (const T*)x.data_ptr(),                      \
                     (const T*)gate.data_ptr(), x.stride(0), gate.stride(0), \
                     sp, state_out.data_ptr<float>(), (T*)y.data_ptr(),      \
                     n_vec, vpr, (int)D, relu)
  SCAN_DTYPES(x.scalar_type(), RUN)
#undef RUN
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return y;
}
