// The join of two transformer blocks and its gradient, for CDNA4 (gfx950):
// the norm on a block's output, its gate, the scaled residual sum and the norm
// before the next block, in one pass over the rows.
// ref semantics: src/models/transformer.h preProcess / postProcess and the
// highway functor of src/tensors/gpu/tensor_operators.cu.
//
//   u = norm_post(x) or x             s = a res + b u
//   h = norm_pre(s)                   a, b = alpha, 1             (no gate)
//                                            alpha, gate          (scale)
//                                            alpha (1-k), k       (highway,
//                                                  k = sigmoid(gate))
//   norm: (v - mean) / sqrt(var + eps) * w (+ bias), or with mean 0 and
//   mean(v^2) for var (rms).
//
// Every row is held in registers in 32 bits by the lanes that work on it:
// each tensor is read once and written once. The variance is summed over
// (v - mean)^2, which costs a second reduction but no second read, and does
// not cancel when the mean is far from 0. h is taken from the 32-bit s, not
// from the rounded one that is stored.
//
// Backward: from x, res, gate and the four saved row statistics u, s and both
// normalised rows are computed again, so that
//   ds = dsum + norm_pre'(dh)    dres = a ds    du = b ds   dx = norm_post'(du)
//   dgate = u ds  or  k (1-k) (u - alpha res) ds
// need no stored intermediate. A lane keeps the columns it works on in all of
// its rows and adds up their parameter gradients in registers; the blocks'
// partial rows are summed by a second kernel in a fixed order (no atomics).
//
// The kernels are instantiated per element type, a source file each.
#pragma once

#include "common.h"
#include "vec.h"

namespace mamd {

enum { kGateNone = 0, kGateChannel = 1, kGateToken = 2 };
// the parameter gradients' rows in a block's partial sums
enum { kPostScale = 0, kPostBias, kPreScale, kPreBias, kGate, kNumParams };

struct NormArgs {
  const void* x;
  const void* res;
  const void* gate;          // null, [D] or [R,D]
  const void* post_scale;    // parameters: [D] or null
  const void* post_bias;
  const void* pre_scale;
  const void* pre_bias;
  int param32;               // parameters are float32 rather than x's type
  int rms, highway;
  float alpha, eps;
  long rows;
  int D;
  int tpr;                   // lanes per row, a power of two
  float* stat;               // [4][rows]: post mean, post 1/dev, pre ..., or null
  // forward
  void* s;
  void* h;
  // backward
  const void* dsum;          // either may be null
  const void* dh;
  void* dx;                  // any of these may be null
  void* dres;
  void* dgate;               // kGateToken only
  float* part;               // [blocks][n_part][D] or null
  int n_part;
  int slot[kNumParams];      // a parameter's row in part, or -1
};

// sums of two values over the lanes of a row, given to all of them. Rows of
// more than a wave meet in LDS; alternating between two buffers makes one
// barrier enough.
struct RowSum {
  float (*buf)[32];
  int tpr, flip;
  __device__ RowSum(float (*b)[32], int t) : buf(b), tpr(t), flip(0) {}
  __device__ __forceinline__ void operator()(float& p, float& q) {
    for (int off = min(tpr, WAVE) >> 1; off > 0; off >>= 1) {
      p += __shfl_xor(p, off, WAVE);
      q += __shfl_xor(q, off, WAVE);
    }
    if (tpr > WAVE) {  // one row per block
      const int nw = tpr / WAVE, wid = threadIdx.x / WAVE;
      if (threadIdx.x % WAVE == 0)
        buf[flip][wid] = p, buf[flip][16 + wid] = q;
      __syncthreads();
      p = q = 0.f;
      for (int i = 0; i < nw; ++i) p += buf[flip][i], q += buf[flip][16 + i];
      flip ^= 1;
    }
  }
};

template <typename T, int VEC>
__device__ __forceinline__ void load_f32(const T* p, int n, float* o) {
  if (n >= VEC) {
    const vec_t<T, VEC> r = load_vec<T, VEC>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = (float)r[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = i < n ? (float)p[i] : 0.f;
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_f32(T* p, int n, const float* o) {
  if (n >= VEC) {
    store_vec<T, VEC>(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) p[i] = (T)o[i];
  }
}

// a parameter vector, whose type may be x's or float32; null: the default
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, int param32, int c,
                                           int n, float dflt, float* o) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = dflt;
  } else if (param32) {
    load_f32<float, VEC>((const float*)p + c, n, o);
  } else {
    load_f32<T, VEC>((const T*)p + c, n, o);
  }
}

// EPT elements per lane in chunks of 16 bytes
template <typename T>
constexpr int vec_of() { return 16 / (int)sizeof(T); }

template <typename T, int EPT, int GATE>
__device__ __forceinline__ void load_gate(const NormArgs& a, long row, int c0,
                                          int step, float* gt) {
  constexpr int VEC = vec_of<T>(), NC = EPT / VEC;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = c0 + i * step, n = a.D - c;
    if constexpr (GATE == kGateToken)
      load_f32<T, VEC>((const T*)a.gate + row * a.D + c, n, gt + i * VEC);
    else
      load_param<T, VEC>(a.gate, a.param32, c, n, 0.f, gt + i * VEC);
  }
}

// coefficients of res and u; k is the highway gate's sigmoid
template <typename T, int GATE>
__device__ __forceinline__ void coefs(const NormArgs& a, float gt, float& ca,
                                      float& cb, float& k, float& k1) {
  ca = a.alpha, cb = 1.f, k = 0.f, k1 = 1.f;
  if constexpr (GATE != kGateNone) {
    if (a.highway) {
      sigmoid2<T>(gt, k, k1);
      ca = a.alpha * k1, cb = k;
    } else {
      cb = gt;
    }
  }
}

// mean and 1/deviation of the elements that exist
template <int EPT, int VEC>
__device__ __forceinline__ void stats(const float* v, int c0, int step, int D,
                                      int rms, float eps, RowSum& sum,
                                      float& mean, float& rstd) {
  float p = 0.f, q = 0.f;
  mean = 0.f;
  if (!rms) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) p += v[i];  // absent elements are 0
    sum(p, q);
    mean = p / D;
  }
  q = p = 0.f;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const float e = v[i] - mean;
    q += c0 + (i / VEC) * step + i % VEC < D ? e * e : 0.f;
  }
  sum(q, p);
  rstd = 1.f / sqrtf(q / D + eps);
}

template <typename T, int EPT, bool POST, bool PRE, int GATE, int MAXT>
__global__ __launch_bounds__(MAXT) void join_fwd_kernel(NormArgs a) {
  constexpr int VEC = vec_of<T>(), NC = EPT / VEC;
  __shared__ float buf[2][32];
  RowSum sum(buf, a.tpr);
  const int lane = threadIdx.x & (a.tpr - 1);
  const int rpb = max((int)blockDim.x / a.tpr, 1);
  const int c0 = lane * VEC, step = a.tpr * VEC;
  for (long r0 = (long)blockIdx.x * rpb; r0 < a.rows;
       r0 += (long)gridDim.x * rpb) {
    long row = r0 + threadIdx.x / a.tpr;
    const bool on = row < a.rows;
    if (!on) row = a.rows - 1;  // its lanes work along and store nothing
    const long base = row * a.D;
    float x[EPT], s[EPT], gt[EPT];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * step;
      load_f32<T, VEC>((const T*)a.x + base + c, a.D - c, x + i * VEC);
      load_f32<T, VEC>((const T*)a.res + base + c, a.D - c, s + i * VEC);
    }
    if constexpr (GATE != kGateNone)
      load_gate<T, EPT, GATE>(a, row, c0, step, gt);
    float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
    if constexpr (POST) {
      stats<EPT, VEC>(x, c0, step, a.D, a.rms, a.eps, sum, m1, r1);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step, n = a.D - c;
        float w[VEC], bb[VEC];
        load_param<T, VEC>(a.post_scale, a.param32, c, n, 1.f, w);
        load_param<T, VEC>(a.post_bias, a.param32, c, n, 0.f, bb);
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          x[i * VEC + v] = (x[i * VEC + v] - m1) * r1 * w[v] + bb[v];
      }
    }
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      float ca, cb, k, k1;
      coefs<T, GATE>(a, GATE ? gt[i] : 0.f, ca, cb, k, k1);
      const bool in = c0 + (i / VEC) * step + i % VEC < a.D;
      s[i] = in ? ca * s[i] + cb * x[i] : 0.f;
    }
    if (on) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step;
        store_f32<T, VEC>((T*)a.s + base + c, a.D - c, s + i * VEC);
      }
    }
    if constexpr (PRE) {
      stats<EPT, VEC>(s, c0, step, a.D, a.rms, a.eps, sum, m2, r2);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step, n = a.D - c;
        float w[VEC], bb[VEC];
        load_param<T, VEC>(a.pre_scale, a.param32, c, n, 1.f, w);
        load_param<T, VEC>(a.pre_bias, a.param32, c, n, 0.f, bb);
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          s[i * VEC + v] = (s[i * VEC + v] - m2) * r2 * w[v] + bb[v];
        if (on) store_f32<T, VEC>((T*)a.h + base + c, n, s + i * VEC);
      }
    }
    if (a.stat && on && lane == 0) {
      a.stat[row] = m1;
      a.stat[a.rows + row] = r1;
      a.stat[2 * a.rows + row] = m2;
      a.stat[3 * a.rows + row] = r2;
    }
  }
}

template <typename T, int EPT, bool POST, bool PRE, int GATE, int MAXT>
__global__ __launch_bounds__(MAXT) void join_bwd_kernel(NormArgs a) {
  constexpr int VEC = vec_of<T>(), NC = EPT / VEC;
  __shared__ float buf[2][32];
  __shared__ float fold[EPT * 256];  // the groups' sums of one parameter
  RowSum sum(buf, a.tpr);
  const int lane = threadIdx.x & (a.tpr - 1);
  const int rpb = max((int)blockDim.x / a.tpr, 1);
  const int c0 = lane * VEC, step = a.tpr * VEC;

  float acc[kNumParams][EPT];  // the unused ones are optimised out
#pragma unroll
  for (int p = 0; p < kNumParams; ++p)
#pragma unroll
    for (int i = 0; i < EPT; ++i) acc[p][i] = 0.f;

  for (long r0 = (long)blockIdx.x * rpb; r0 < a.rows;
       r0 += (long)gridDim.x * rpb) {
    long row = r0 + threadIdx.x / a.tpr;
    const bool on = row < a.rows;
    if (!on) row = a.rows - 1;
    const long base = row * a.D;
    float x[EPT], rs[EPT], ds[EPT], dh[EPT], gt[EPT];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * step, n = a.D - c;
      if constexpr (POST || PRE || GATE != kGateNone)
        load_f32<T, VEC>((const T*)a.x + base + c, n, x + i * VEC);
      if constexpr (PRE || GATE != kGateNone)
        load_f32<T, VEC>((const T*)a.res + base + c, n, rs + i * VEC);
      if (a.dsum) {
        load_f32<T, VEC>((const T*)a.dsum + base + c, n, ds + i * VEC);
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) ds[i * VEC + v] = 0.f;
      }
      if constexpr (PRE) {
        if (a.dh) {
          load_f32<T, VEC>((const T*)a.dh + base + c, n, dh + i * VEC);
        } else {
#pragma unroll
          for (int v = 0; v < VEC; ++v) dh[i * VEC + v] = 0.f;
        }
      }
    }
    if constexpr (GATE != kGateNone)
      load_gate<T, EPT, GATE>(a, row, c0, step, gt);
    const float m1 = a.stat[row], r1 = a.stat[a.rows + row];
    const float m2 = a.stat[2 * a.rows + row], r2 = a.stat[3 * a.rows + row];
    if (!on) {  // nothing may reach the parameter sums
#pragma unroll
      for (int i = 0; i < EPT; ++i) ds[i] = dh[i] = 0.f;
    }
    // x becomes the normalised row
    float u[EPT];
    if constexpr (POST) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step, n = a.D - c;
        float w[VEC], bb[VEC];
        load_param<T, VEC>(a.post_scale, a.param32, c, n, 1.f, w);
        load_param<T, VEC>(a.post_bias, a.param32, c, n, 0.f, bb);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const int e = i * VEC + v;
          x[e] = (x[e] - m1) * r1;
          u[e] = x[e] * w[v] + bb[v];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) u[i] = x[i];
    }
    if constexpr (PRE) {
      float sh[EPT], p = 0.f, q = 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step;
        float w[VEC];
        load_param<T, VEC>(a.pre_scale, a.param32, c, a.D - c, 1.f, w);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const int e = i * VEC + v;
          float ca, cb, k, k1;
          coefs<T, GATE>(a, GATE ? gt[e] : 0.f, ca, cb, k, k1);
          sh[e] = (ca * rs[e] + cb * u[e] - m2) * r2;
          acc[kPreScale][e] += dh[e] * sh[e];
          acc[kPreBias][e] += dh[e];
          dh[e] *= w[v];  // 0 where there is no element
          p += dh[e];
          q += dh[e] * sh[e];
        }
      }
      sum(p, q);
      p = a.rms ? 0.f : p / a.D;
      q /= a.D;
#pragma unroll
      for (int i = 0; i < EPT; ++i) ds[i] += r2 * (dh[i] - p - sh[i] * q);
    }
    float p = 0.f, q = 0.f, du[EPT];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = c0 + i * step, n = a.D - c;
      float w[VEC], dr[VEC], dg[VEC];
      if constexpr (POST)
        load_param<T, VEC>(a.post_scale, a.param32, c, n, 1.f, w);
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const int e = i * VEC + v;
        float ca, cb, k, k1;
        coefs<T, GATE>(a, GATE ? gt[e] : 0.f, ca, cb, k, k1);
        const float d = c + v < a.D ? ds[e] : 0.f;
        dr[v] = ca * d;
        du[e] = cb * d;
        if constexpr (GATE != kGateNone) {
          dg[v] = (a.highway ? k * k1 * (u[e] - a.alpha * rs[e]) : u[e]) * d;
          // a row of another lane group's past the end adds nothing
          if (!on) dg[v] = 0.f;
          if constexpr (GATE == kGateChannel) acc[kGate][e] += dg[v];
        }
        if constexpr (POST) {
          acc[kPostScale][e] += on ? du[e] * x[e] : 0.f;
          acc[kPostBias][e] += on ? du[e] : 0.f;
          du[e] *= w[v];
          p += du[e];
          q += du[e] * x[e];
        }
      }
      if (on && a.dres) store_f32<T, VEC>((T*)a.dres + base + c, n, dr);
      if constexpr (GATE == kGateToken)
        if (on && a.dgate) store_f32<T, VEC>((T*)a.dgate + base + c, n, dg);
    }
    if constexpr (POST) {
      sum(p, q);
      p = a.rms ? 0.f : p / a.D;
      q /= a.D;
#pragma unroll
      for (int i = 0; i < EPT; ++i) du[i] = r1 * (du[i] - p - x[i] * q);
    }
    if (on && a.dx) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = c0 + i * step;
        store_f32<T, VEC>((T*)a.dx + base + c, a.D - c, du + i * VEC);
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + (size_t)blockIdx.x * a.n_part * a.D;
#pragma unroll
  for (int p = 0; p < kNumParams; ++p) {
    if (a.slot[p] < 0) continue;
    float* out = part + (size_t)a.slot[p] * a.D;
    if (rpb == 1) {
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int c = c0 + (i / VEC) * step + i % VEC;
        if (c < a.D) out[c] = acc[p][i];
      }
    } else {  // blockDim.x is 256 here
      __syncthreads();
#pragma unroll
      for (int i = 0; i < EPT; ++i)
        fold[i * 256 + threadIdx.x] = acc[p][i];
      __syncthreads();
      if (threadIdx.x < a.tpr) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          const int c = c0 + (i / VEC) * step + i % VEC;
          float t = 0.f;
          for (int g = 0; g < rpb; ++g)
            t += fold[i * 256 + g * a.tpr + threadIdx.x];
          if (c < a.D) out[c] = t;
        }
      }
    }
  }
}

struct NormPlan {
  NormArgs a{};
  int gate_mode = kGateNone;
  int ept = 8, threads = 256, rpb = 1;
};

#define GATES(T, EPT, POST, PRE, MAXT, FN)                              \
  if (pl.gate_mode == kGateNone) { FN(T, EPT, POST, PRE, kGateNone, MAXT); }      \
  else if (pl.gate_mode == kGateChannel) { FN(T, EPT, POST, PRE, kGateChannel, MAXT); } \
  else { FN(T, EPT, POST, PRE, kGateToken, MAXT); }
#define SIDES(T, EPT, MAXT, FN)                                         \
  if (a.post_scale && a.pre_scale) { GATES(T, EPT, true, true, MAXT, FN) }        \
  else if (a.post_scale) { GATES(T, EPT, true, false, MAXT, FN) }       \
  else if (a.pre_scale) { GATES(T, EPT, false, true, MAXT, FN) }        \
  else { GATES(T, EPT, false, false, MAXT, FN) }
#define WIDTHS(T, FN)                                                   \
  if (pl.ept == 8) { SIDES(T, 8, 512, FN) }                             \
  else if (pl.threads <= 512) { SIDES(T, 16, 512, FN) }                 \
  else { SIDES(T, 16, 1024, FN) }

template <typename T>
void join_fwd_launch(const NormPlan& pl, unsigned grid, hipStream_t stream) {
  const NormArgs& a = pl.a;
#define RUN(T, EPT, POST, PRE, GATE, MAXT)                                   \
  hipLaunchKernelGGL((join_fwd_kernel<T, EPT, POST, PRE, GATE, MAXT>),       \
                     dim3(grid), dim3(pl.threads), 0, stream, a)
  WIDTHS(T, RUN)
#undef RUN
}

template <typename T>
void join_bwd_launch(const NormPlan& pl, unsigned grid, hipStream_t stream) {
  const NormArgs& a = pl.a;
#define RUN(T, EPT, POST, PRE, GATE, MAXT)                                   \
  hipLaunchKernelGGL((join_bwd_kernel<T, EPT, POST, PRE, GATE, MAXT>),       \
                     dim3(grid), dim3(pl.threads), 0, stream, a)
  WIDTHS(T, RUN)
#undef RUN
}

#undef WIDTHS
#undef SIDES
#undef GATES

}  // namespace mamd
