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
// What bounds it: bytes. 65536 x 1024 bf16 with two layer norms and a channel's
// factor: forward 4 tensors, backward 6, 284 us for both, 4.7 TB/s where a copy
// of 2 GB runs at 4.9 (kernels in a profile, at the median: 110, and 197 + 13
// for the parameter sums); a factor per token 355 us (4.9), a highway per token
// 374 (4.7). What brought it there: parameters and the next row kept in
// registers, rows walked by as many blocks as the GPU holds at once (forward
// 250 -> 107, backward 393 -> 190) and two rows a block in the backward pass
// (-> 173, then with four sums). float32 parameters beside 16-bit rows are read
// again for every row: 332 us for 284.
// Rows of 4097 columns on have 16 elements a lane, and their backward kernels
// spill where sums and operands are many, by the compiler's report: up to 8192
// columns only with both norms (bf16: 4 registers with a factor or a factor per
// token, 46 and 75 with highways; fp32: 6 without a gate, 72 - 155 with one)
// and, in fp32, 8 for a highway with one norm; rms norms without biases, whose
// kernel has 32 sums fewer to hold, in highways alone (10 - 20). From 8193
// columns on lanes have 128 registers and nearly all forms with a pre norm or a
// gate spill (bf16 12 - 213, fp32 8 - 218). Kernels, bf16, layer norms and rms:
// 2048 x 8192 61 and 48 us (75 and 48 with a factor), 2048 x 16384 with a
// factor 362 and 221.
//
// The kernels are instantiated per element type, a source file each.
#pragma once

#include <atomic>

#include "common.h"
#include "vec.h"

namespace mamd {

// gates: per channel or per token, a factor or a highway's logit
enum { kNone = 0, kScaleCh, kScaleTok, kHighCh, kHighTok };
constexpr bool is_highway(int g) { return g == kHighCh || g == kHighTok; }
constexpr bool is_channel(int g) { return g == kScaleCh || g == kHighCh; }
constexpr bool is_token(int g) { return g == kScaleTok || g == kHighTok; }

// Sums over rows that the parameter gradients are made of, xh and sh the
// normalised rows (xh = x without a post norm):
//   dpre_scale = P1, dpre_bias = P0, dpost_scale = b S1, dpost_bias = b S0,
//   dgate = S2, or w1 S1 without a post bias   (scale, per channel)
//           k (1-k) S2                         (highway, per channel)
// since b and w1 do not change along the rows. S2 is the sum of u ds, or of
// (u - alpha res) ds: whole sums of xh ds, ds and res ds, put together
// afterwards, cancel where a bias takes back a channel that the norm makes
// large (1 - 3 % of the gradient was wrong, now 0.08 %), or where u and res
// have a common mean (4096 rows of deviation 1 around 300: 1e-3 of it, now
// 2e-7). With a gate per token S1 and S0 take b inside.
enum { kS1 = 0, kS0, kS2, kP1, kP0, kNumSums };

struct NormArgs {
  const void* x;
  const void* res;           // null: zeros
  const void* gate;          // null, [D] or [R,D]
  const void* post_scale;    // parameters: [D] or null
  const void* post_bias;
  const void* pre_scale;
  const void* pre_bias;
  int param32;               // parameters are float32 rather than x's type
  int rms;
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
  void* dgate;               // per token
  float* part;               // [blocks][n_part][D] or null
  int n_part;
  int slot[kNumSums];        // a sum's row in part, or -1
};

// How a row's lanes are placed: some lanes of a wave, one wave, two of a
// block's four waves, or a block.
enum { kPartWave = 0, kWave = 1, kPair = 2, kBlock = 3 };
// lane groups that may be without a row while others of their wave or block
// still have one
constexpr bool may_idle(int place) { return place == kPartWave || place == kPair; }

// sum over a wave in a fixed order, in all lanes: 4 steps inside rows of 16
// lanes and 2 between them, all of them modifiers of an add
__device__ __forceinline__ float dpp_sum(float v) {
#define STEP(CTRL, ROWS)                                                  \
  v += __int_as_float(__builtin_amdgcn_update_dpp(                        \
      0, __float_as_int(v), CTRL, ROWS, 0xf, true))
  STEP(0x111, 0xf);  // row_shr:1
  STEP(0x112, 0xf);
  STEP(0x114, 0xf);
  STEP(0x118, 0xf);
  STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// sums of two values over the lanes of a row, given to all of them. The waves
// of a block meet in LDS; alternating between two buffers makes one barrier
// enough.
template <int PLACE>
struct RowSum {
  float (*buf)[32];
  int tpr, flip;
  __device__ RowSum(float (*b)[32], int t) : buf(b), tpr(t), flip(0) {}
  __device__ __forceinline__ void operator()(float& p, float& q) {
    if constexpr (PLACE == kPartWave) {
      for (int off = tpr >> 1; off > 0; off >>= 1) {
        p += __shfl_xor(p, off, WAVE);
        q += __shfl_xor(q, off, WAVE);
      }
    } else {
      p = dpp_sum(p);
      q = dpp_sum(q);
    }
    if constexpr (PLACE == kPair || PLACE == kBlock) {
      const int wid = threadIdx.x / WAVE;
      if (threadIdx.x % WAVE == 0)
        buf[flip][wid] = p, buf[flip][16 + wid] = q;
      __syncthreads();
      if constexpr (PLACE == kPair) {
        const float* w = &buf[flip][wid & ~1];
        p = w[0] + w[1], q = w[16] + w[17];
      } else {
        const int nw = tpr / WAVE;
        p = q = 0.f;
        for (int i = 0; i < nw; ++i) p += buf[flip][i], q += buf[flip][16 + i];
      }
      flip ^= 1;
    }
  }
  __device__ __forceinline__ void operator()(float& p) {
    if constexpr (PLACE == kWave) {
      p = dpp_sum(p);
    } else {
      float q = 0.f;
      (*this)(p, q);
    }
  }
};

// A lane's columns: NC vectors of VEC, `step` apart. A vector that would pass
// the row's end moves back to the row's last VEC columns: it computes what its
// neighbour computes and writes the same values there, but the columns that it
// has twice (those before `first`) stay out of every sum.
template <int VEC, int NC>
struct Columns {
  int at[NC], first[NC];
  __device__ __forceinline__ Columns(int lane, int tpr, int D) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      first[i] = (lane + i * tpr) * VEC;
      at[i] = min(first[i], D - VEC);
    }
  }
  __device__ __forceinline__ bool own(int e) const {
    return at[e / VEC] + e % VEC >= first[e / VEC];
  }
  __device__ __forceinline__ bool any(int i, int D) const {
    return first[i] < D;
  }
};

template <typename T, int VEC, int NC>
struct RawRow {
  vec_t<T, VEC> r[NC];
  __device__ __forceinline__ void load(const T* p,
                                       const Columns<VEC, NC>& c) {
#pragma unroll
    for (int i = 0; i < NC; ++i) r[i] = load_vec<T, VEC>(p + c.at[i]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NC; ++i) r[i] = {};
  }
  __device__ __forceinline__ float operator[](int e) const {
    return (float)r[e / VEC][e % VEC];
  }
};

template <typename V>
__device__ __forceinline__ V opaque(V v) {
  if constexpr (sizeof(V) % 4 == 0) {
    unsigned w[sizeof(V) / 4];
    __builtin_memcpy(w, &v, sizeof(V));
#pragma unroll
    for (unsigned& x : w) asm("" : "+v"(x));
    __builtin_memcpy(&v, w, sizeof(V));
  }
  return v;
}

// A parameter vector's columns. KEEP: those of x's type stay in registers, in
// that type, over the rows of a block (the empty asm keeps the compiler from
// holding their 32-bit values instead, twice the registers). Others - float32
// ones beside 16-bit rows - are read again for each row, from L1 or L2.
template <typename T, int VEC, int NC, bool KEEP>
struct Param {
  const void* p;
  int wide;
  float dflt;
  RawRow<T, VEC, KEEP ? NC : 1> raw;
  __device__ __forceinline__ Param(const void* p_, int param32, float d,
                                   const Columns<VEC, NC>& c)
      : p(p_), wide(param32 && sizeof(T) != 4), dflt(d) {
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) raw.r[i][v] = (T)d;
      if (p && !wide) raw.load((const T*)p, c);
    }
  }
  __device__ __forceinline__ void get(const Columns<VEC, NC>& c,
                                      float o[VEC * NC]) const {
    if (KEEP && !(sizeof(T) != 4 && wide)) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const vec_t<T, VEC> r = opaque(raw.r[KEEP ? i : 0]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[i * VEC + v] = (float)r[v];
      }
    } else if (!p) {
#pragma unroll
      for (int e = 0; e < VEC * NC; ++e) o[e] = dflt;
    } else if (sizeof(T) != 4 && wide) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const vec_t<float, VEC> w =
            load_vec<float, VEC>((const float*)p + c.at[i]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[i * VEC + v] = w[v];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const vec_t<T, VEC> w = load_vec<T, VEC>((const T*)p + c.at[i]);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[i * VEC + v] = (float)w[v];
      }
    }
  }
};

// coefficients of res and u; k is the highway gate's sigmoid
template <typename T, int GATE>
__device__ __forceinline__ void coefs(float alpha, float gt, float& ca,
                                      float& cb, float& k1) {
  ca = alpha, cb = 1.f, k1 = 1.f;
  if constexpr (is_highway(GATE)) {
    sigmoid2<T>(gt, cb, k1);
    ca = alpha * k1;
  } else if constexpr (GATE != kNone) {
    cb = gt;
  }
}

// mean and 1/deviation of a row
template <int VEC, int NC, int PLACE>
__device__ __forceinline__ void stats(const float* v,
                                      const Columns<VEC, NC>& c,
                                      float inv_d, int rms, float eps,
                                      RowSum<PLACE>& sum,
                                      float& mean, float& rstd) {
  mean = 0.f;
  if (!rms) {
    float p = 0.f;
#pragma unroll
    for (int e = 0; e < VEC * NC; ++e) p += c.own(e) ? v[e] : 0.f;
    sum(p);
    mean = p * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < VEC * NC; ++e) {
    const float d = c.own(e) ? v[e] - mean : 0.f;
    q += d * d;
  }
  sum(q);
  rstd = rsqrtf(q * inv_d + eps);
}

// the rows of a lane group: row, row + stride, ...; row0 is its block's first
template <int PLACE>
struct Rows {
  long row, row0, stride;
  int lane;
  __device__ __forceinline__ Rows(const NormArgs& a) {
    if constexpr (PLACE == kBlock) {
      lane = threadIdx.x;
      row = row0 = blockIdx.x;
      stride = gridDim.x;
    } else {
      const int rpb = blockDim.x / a.tpr;
      lane = threadIdx.x & (a.tpr - 1);
      int group = threadIdx.x / a.tpr;
      if constexpr (PLACE != kPartWave)
        group = __builtin_amdgcn_readfirstlane(group);
      row0 = (long)blockIdx.x * rpb;
      row = row0 + group;
      stride = (long)gridDim.x * rpb;
    }
  }
};

// Lane groups without a row (at the end of the last block) work on the last
// row, in the backward pass on zeros, and store nothing; a row's sums never
// leave its lane group.
template <typename T, int VEC, int EPT, int PLACE, bool POST, bool PRE,
          int GATE, int MAXT>
__global__ __launch_bounds__(MAXT) void join_fwd_kernel(NormArgs a) {
  constexpr int NC = EPT / VEC;
  // blocks of 1024 have 128 registers a lane: parameters are read again for
  // each row and nothing is fetched ahead
  constexpr bool KEEP = MAXT <= 512;
  using Raw = RawRow<T, VEC, NC>;
  __shared__ float buf[2][32];
  RowSum<PLACE> sum(buf, a.tpr);
  const float inv_d = 1.f / (float)a.D;
  const Rows<PLACE> it(a);
  const Columns<VEC, NC> col(it.lane, a.tpr, a.D);
  const Param<T, VEC, NC, KEEP> w1(POST ? a.post_scale : nullptr, a.param32, 1.f,
                             col);
  const Param<T, VEC, NC, KEEP> b1(POST ? a.post_bias : nullptr, a.param32, 0.f,
                             col);
  const Param<T, VEC, NC, KEEP> w2(PRE ? a.pre_scale : nullptr, a.param32, 1.f, col);
  const Param<T, VEC, NC, KEEP> b2(PRE ? a.pre_bias : nullptr, a.param32, 0.f, col);
  const Param<T, VEC, NC, KEEP> gp(is_channel(GATE) ? a.gate : nullptr,
                             a.param32, 0.f, col);

  Raw xr, rr, gr;
  auto fetch = [&](long row) __attribute__((always_inline)) {
    const long base = min(row, a.rows - 1) * a.D;
    xr.load((const T*)a.x + base, col);
    if (a.res) rr.load((const T*)a.res + base, col);
    if constexpr (is_token(GATE)) gr.load((const T*)a.gate + base, col);
  };
  rr.zero();
  if (KEEP) fetch(it.row);
  // the same number of turns for all lanes of a wave
  for (long r0 = 0, n = (a.rows + it.stride - 1) / it.stride; r0 < n; ++r0) {
    const long row = it.row + r0 * it.stride;
    // waves that meet at barriers work on one row
    if (PLACE != kPartWave && row >= a.rows) break;
    if (!KEEP) fetch(row);
    const bool on = !may_idle(PLACE) || row < a.rows;
    const long base = row * a.D;
    float x[EPT], s[EPT], gt[EPT], w[EPT], bb[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      x[e] = xr[e];
      s[e] = rr[e];
      gt[e] = is_token(GATE) ? gr[e] : 0.f;
    }
    if (KEEP && r0 + 1 < n) fetch(row + it.stride);
    if constexpr (is_channel(GATE)) gp.get(col, gt);
    float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
    if constexpr (POST) {
      stats<VEC, NC, PLACE>(x, col, inv_d, a.rms, a.eps, sum, m1, r1);
      w1.get(col, w);
      b1.get(col, bb);
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = (x[e] - m1) * r1 * w[e] + bb[e];
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      float ca, cb, k1;
      coefs<T, GATE>(a.alpha, gt[e], ca, cb, k1);
      s[e] = ca * s[e] + cb * x[e];
    }
    if (on) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (col.any(i, a.D))
          store_vec<T, VEC>((T*)a.s + base + col.at[i], s + i * VEC);
    }
    if constexpr (PRE) {
      stats<VEC, NC, PLACE>(s, col, inv_d, a.rms, a.eps, sum, m2, r2);
      w2.get(col, w);
      b2.get(col, bb);
#pragma unroll
      for (int e = 0; e < EPT; ++e) s[e] = (s[e] - m2) * r2 * w[e] + bb[e];
      if (on) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
          if (col.any(i, a.D))
            store_vec<T, VEC>((T*)a.h + base + col.at[i], s + i * VEC);
      }
    }
    if (a.stat && on && it.lane == 0) {
      a.stat[row] = m1;
      a.stat[a.rows + row] = r1;
      a.stat[2 * a.rows + row] = m2;
      a.stat[3 * a.rows + row] = r2;
    }
  }
}

// LEAN: rms norms without biases, which need neither the mean nor the sums of
// gradients alone.
template <typename T, int VEC, int EPT, int PLACE, bool POST, bool PRE,
          int GATE, int MAXT, bool LEAN>
__global__ __launch_bounds__(MAXT) void join_bwd_kernel(NormArgs a) {
  constexpr int NC = EPT / VEC;
  // blocks of 1024 have 128 registers a lane: parameters are read again for
  // each row and nothing is fetched ahead
  constexpr bool KEEP = MAXT <= 512;
  // Rows of 16 elements a lane leave no registers for the next row's, except
  // where the sums and the operands are few. rms, this kernel alone, with the
  // fetch ahead and without: 2048 x 8192 bf16 no gate 37.6 us for 40.5 with a
  // pre norm and 47.4 for 47.1 with both, 2048 x 6000 37.8 for 38.9, with a
  // factor 38.9 for 39.9 (44.6 for 43.8 at 8192 and a pre norm). Gates per
  // token gain nothing, and fp32 spills: a whole pass of 4096 x 6000 with a
  // factor and both norms takes 303 us for 199.
  constexpr bool FEW =
      LEAN && sizeof(T) == 2 && (GATE == kNone || GATE == kScaleCh);
  constexpr bool AHEAD = KEEP && (!(PLACE == kBlock && EPT == 16) || FEW);
  using Raw = RawRow<T, VEC, NC>;
  __shared__ float buf[2][32];
  // the lane groups' sums of one parameter
  __shared__ float fold[PLACE == kBlock ? 1 : EPT * 256];
  RowSum<PLACE> sum(buf, a.tpr);
  const float inv_d = 1.f / (float)a.D;
  const Rows<PLACE> it(a);
  const Columns<VEC, NC> col(it.lane, a.tpr, a.D);
  const Param<T, VEC, NC, KEEP> w1(POST ? a.post_scale : nullptr, a.param32, 1.f,
                             col);
  const Param<T, VEC, NC, KEEP> b1(POST && !LEAN ? a.post_bias : nullptr, a.param32, 0.f,
                             col);
  const Param<T, VEC, NC, KEEP> w2(PRE ? a.pre_scale : nullptr, a.param32, 1.f, col);
  const Param<T, VEC, NC, KEEP> gp(is_channel(GATE) ? a.gate : nullptr,
                             a.param32, 0.f, col);
  // s and u are needed by the next norm and by the gate
  constexpr bool NEED = PRE || GATE != kNone;
  // A factor's S2 takes a fifth sum and its operands, and the registers for a
  // third wave on each SIMD. In LDS, each lane's to itself, and apart from the
  // rest of a row (nothing is moved over the two barriers) it leaves them:
  // whole passes of 131072 x 512 bf16 281 us for 311, 262144 x 200 282 for 329;
  // where 16 elements a lane spill, 2048 x 8192 117 for 127 and 2048 x 16384
  // 462 for 552. Rows over two waves (164 registers, 3 waves) and blocks of 8
  // elements a lane are better off with registers: 65536 x 1024 283 for 291,
  // 8192 x 4096 174 for 183.
  constexpr bool FACTOR = GATE == kScaleCh && POST && !LEAN;
  constexpr bool IN_LDS = FACTOR && (PLACE <= kWave || EPT == 16);
  constexpr int QUAD = EPT % 4 == 0 ? 4 : 1;
  __shared__ vec_t<float, QUAD> factor[IN_LDS ? EPT / QUAD * MAXT : 1];
  if constexpr (IN_LDS) {
#pragma unroll
    for (int i = 0; i < EPT / QUAD; ++i) factor[i * MAXT + threadIdx.x] = {};
  }

  float acc[kNumSums][EPT];  // the unused ones are optimised out
#pragma unroll
  for (int p = 0; p < kNumSums; ++p)
#pragma unroll
    for (int e = 0; e < EPT; ++e) acc[p][e] = 0.f;

  Raw xr, rr, dr, hr, gr;
  float st[4];
  rr.zero();
  auto fetch = [&](long row) __attribute__((always_inline)) {
    if (may_idle(PLACE) && row >= a.rows) {  // zeros add nothing to the sums
      xr.zero(), rr.zero(), dr.zero(), hr.zero(), gr.zero();
#pragma unroll
      for (int i = 0; i < 4; ++i) st[i] = 0.f;
      return;
    }
    row = min(row, a.rows - 1);
    const long base = row * a.D;
    if constexpr (POST || NEED) xr.load((const T*)a.x + base, col);
    if (NEED && a.res) rr.load((const T*)a.res + base, col);
    dr.zero();
    hr.zero();
    if (a.dsum) dr.load((const T*)a.dsum + base, col);
    if (PRE && a.dh) hr.load((const T*)a.dh + base, col);
    if constexpr (is_token(GATE)) gr.load((const T*)a.gate + base, col);
#pragma unroll
    for (int i = 0; i < 4; ++i) st[i] = a.stat[i * a.rows + row];
  };
  if (AHEAD) fetch(it.row);
  for (long r0 = 0, n = (a.rows + it.stride - 1) / it.stride; r0 < n; ++r0) {
    const long row = it.row + r0 * it.stride;
    // waves that meet at barriers leave together
    if ((PLACE == kPair ? it.row0 + r0 * it.stride : row) >= a.rows &&
        PLACE != kPartWave)
      break;
    if (!AHEAD) fetch(row);
    const bool on = !may_idle(PLACE) || row < a.rows;
    const long base = row * a.D;
    // this row, 16-bit values kept as they are until they are used
    const Raw rc = rr, dc = dr, hc = hr, gc = gr;
    const float m1 = LEAN ? 0.f : st[0], r1 = st[1];
    const float m2 = LEAN ? 0.f : st[2], r2 = st[3];
    float x[EPT], ds[EPT], w[EPT], bb[EPT], gt[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e)  // the normalised row
      x[e] = POST ? (xr[e] - m1) * r1 : NEED ? xr[e] : 0.f;
    if (AHEAD && r0 + 1 < n) fetch(row + it.stride);
    auto gates = [&]() __attribute__((always_inline)) {
      if constexpr (is_channel(GATE)) gp.get(col, gt);
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        if constexpr (!is_channel(GATE)) gt[e] = is_token(GATE) ? gc[e] : 0.f;
    };
    auto bias = [&](float o[EPT]) __attribute__((always_inline)) {
      if constexpr (LEAN) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] = 0.f;
      } else {
        b1.get(col, o);
      }
    };
    auto row_sums = [&](float& p, float& q) __attribute__((always_inline)) {
      if constexpr (LEAN) {
        sum(q);
        p = 0.f;
      } else {
        sum(p, q);
        p = a.rms ? 0.f : p * inv_d;
      }
      q *= inv_d;
    };
    if constexpr (PRE) {
      float sh[EPT], gh[EPT], p = 0.f, q = 0.f;
      if constexpr (POST) w1.get(col, w), bias(bb);
      gates();
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        float ca, cb, k1;
        coefs<T, GATE>(a.alpha, gt[e], ca, cb, k1);
        const float u = POST ? x[e] * w[e] + bb[e] : x[e];
        sh[e] = (ca * rc[e] + cb * u - m2) * r2;
      }
      w2.get(col, w);
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        const float g = hc[e];
        acc[kP1][e] += g * sh[e];
        if (!LEAN) acc[kP0][e] += g;
        gh[e] = g * w[e];
        p += col.own(e) ? gh[e] : 0.f;
        q += col.own(e) ? gh[e] * sh[e] : 0.f;
      }
      row_sums(p, q);
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        ds[e] = dc[e] + r2 * (gh[e] - p - sh[e] * q);
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e) ds[e] = dc[e];
    }
    if constexpr (IN_LDS) {
      __builtin_amdgcn_sched_barrier(0);
      w1.get(col, w);
      bias(bb);
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        factor[e / QUAD * MAXT + threadIdx.x][e % QUAD] +=
            (x[e] * w[e] + bb[e]) * ds[e];
      __builtin_amdgcn_sched_barrier(0);
    }
    float p = 0.f, q = 0.f, dr_[EPT];
    gates();
    if constexpr (POST) w1.get(col, w);
    // the terms of the gate's gradient are needed one by one
    constexpr bool TERM = is_token(GATE) || GATE == kHighCh ||
                          (FACTOR && !IN_LDS);
    if constexpr (POST && TERM) bias(bb);
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      float ca, cb, k1;
      coefs<T, GATE>(a.alpha, gt[e], ca, cb, k1);
      const float d = ds[e];
      dr_[e] = ca * d;   // the gradient of res
      ds[e] = cb * d;    // and of u
      if constexpr (GATE == kScaleCh || POST) {
        const float t = is_channel(GATE) ? d : ds[e];
        acc[kS1][e] += t * x[e];
        if (!LEAN) acc[kS0][e] += t;
      }
      if constexpr (TERM) {
        const float u = POST ? x[e] * w[e] + bb[e] : x[e];
        const float du = is_highway(GATE) ? u - a.alpha * rc[e] : u;
        if constexpr (is_channel(GATE)) acc[kS2][e] += du * d;
        else gt[e] = (is_highway(GATE) ? cb * k1 * du : du) * d;
      }
      if constexpr (POST) {
        ds[e] *= w[e];
        p += col.own(e) ? ds[e] : 0.f;
        q += col.own(e) ? ds[e] * x[e] : 0.f;
      }
    }
    auto put = [&](void* out, const float* v) __attribute__((always_inline)) {
      if (!on || !out) return;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (col.any(i, a.D))
          store_vec<T, VEC>((T*)out + base + col.at[i], v + i * VEC);
    };
    put(a.dres, dr_);
    if constexpr (is_token(GATE)) put(a.dgate, gt);
    if constexpr (POST) {
      row_sums(p, q);
#pragma unroll
      for (int e = 0; e < EPT; ++e) ds[e] = r1 * (ds[e] - p - x[e] * q);
    }
    put(a.dx, ds);
  }
  if (!a.part) return;
  if constexpr (IN_LDS) {
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      acc[kS2][e] = factor[e / QUAD * MAXT + threadIdx.x][e % QUAD];
  }
  float* part = a.part + (size_t)blockIdx.x * a.n_part * a.D;
#pragma unroll
  for (int p = 0; p < kNumSums; ++p) {
    if (a.slot[p] < 0) continue;
    float* out = part + (size_t)a.slot[p] * a.D;
    if constexpr (PLACE == kBlock) {
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        if (col.own(e)) out[col.at[e / VEC] + e % VEC] = acc[p][e];
    } else {  // blockDim.x is 256
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        fold[e * 256 + threadIdx.x] = acc[p][e];
      __syncthreads();
      if (threadIdx.x < a.tpr) {
        const int groups = 256 / a.tpr;
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
          float t = 0.f;
          for (int g = 0; g < groups; ++g)
            t += fold[e * 256 + g * a.tpr + threadIdx.x];
          if (col.own(e)) out[col.at[e / VEC] + e % VEC] = t;
        }
      }
    }
  }
}

struct NormPlan {
  NormArgs a{};
  int gate = kNone;
  int ept = 8, place = kWave, threads = 256, rpb = 1;
};

#define GATES(T, VEC, EPT, PLACE, POST, PRE, MAXT, FN)                    \
  switch (pl.gate) {                                                      \
    case kNone: FN(T, VEC, EPT, PLACE, POST, PRE, kNone, MAXT)            \
    case kScaleCh: FN(T, VEC, EPT, PLACE, POST, PRE, kScaleCh, MAXT)      \
    case kScaleTok: FN(T, VEC, EPT, PLACE, POST, PRE, kScaleTok, MAXT)    \
    case kHighCh: FN(T, VEC, EPT, PLACE, POST, PRE, kHighCh, MAXT)        \
    default: FN(T, VEC, EPT, PLACE, POST, PRE, kHighTok, MAXT)            \
  }
#define SIDES(T, VEC, EPT, PLACE, MAXT, FN)                               \
  if (a.post_scale && a.pre_scale) {                                      \
    GATES(T, VEC, EPT, PLACE, true, true, MAXT, FN)                       \
  } else if (a.post_scale) {                                              \
    GATES(T, VEC, EPT, PLACE, true, false, MAXT, FN)                      \
  } else if (a.pre_scale) {                                               \
    GATES(T, VEC, EPT, PLACE, false, true, MAXT, FN)                      \
  } else {                                                                \
    GATES(T, VEC, EPT, PLACE, false, false, MAXT, FN)                     \
  }
// The widths' kernels that both passes have, and those of one of them.
#define NARROW(T, FN)                                                     \
  constexpr int V = 16 / (int)sizeof(T);                                  \
  if (pl.ept == 1) {                                                      \
    SIDES(T, 1, 1, kPartWave, 256, FN)                                    \
  } else if (pl.place == kPartWave) {                                     \
    SIDES(T, V, 8, kPartWave, 256, FN)                                    \
  } else if (pl.place == kWave && pl.ept == 8) {                          \
    SIDES(T, V, 8, kWave, 256, FN)                                        \
  }
#define WIDE(T, FN)                                                       \
  if (pl.place == kBlock && pl.ept == 8) {                                \
    SIDES(T, V, 8, kBlock, 512, FN)                                       \
  } else if (pl.place == kBlock && pl.threads <= 512) {                   \
    SIDES(T, V, 16, kBlock, 512, FN)                                      \
  } else if (pl.place == kBlock) {                                        \
    SIDES(T, V, 16, kBlock, 1024, FN)                                     \
  }
#define FWD_WIDTHS(T, FN)                                                 \
  NARROW(T, FN) else if (pl.place == kWave) {                             \
    if constexpr (sizeof(T) == 2) { SIDES(T, V, 16, kWave, 256, FN) }     \
  } else WIDE(T, FN)
#define BWD_WIDTHS(T, FN)                                                 \
  NARROW(T, FN) else if (pl.place == kPair) {                             \
    SIDES(T, V, 8, kPair, 256, FN)                                        \
  } else WIDE(T, FN)

// blocks of a kernel that a CU holds at once, asked for once per block size
template <auto KERNEL>
int resident(int threads) {
  static std::atomic<int> known[11];  // by log2(threads)
  std::atomic<int>& k = known[__builtin_ctz((unsigned)threads)];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
            &n, reinterpret_cast<const void*>(KERNEL), threads, 0) !=
            hipSuccess || n < 1)
      n = 1;
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}

// grid == 0: nothing is launched, the blocks that a CU holds are returned.
// 0 is returned where there is no kernel for the plan.
template <typename T>
int join_fwd_launch(const NormPlan& pl, unsigned grid, hipStream_t stream) {
  const NormArgs& a = pl.a;
#define RUN(T, VEC, EPT, PLACE, POST, PRE, GATE, MAXT)                       \
  {                                                                          \
    constexpr auto kernel =                                                  \
        &join_fwd_kernel<T, VEC, EPT, PLACE, POST, PRE, GATE, MAXT>;         \
    if (grid == 0) return resident<kernel>(pl.threads);                      \
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(pl.threads), 0, stream, a);  \
    return 1;                                                                \
  }
  FWD_WIDTHS(T, RUN)
#undef RUN
  return 0;
}

template <typename T>
int join_bwd_launch(const NormPlan& pl, unsigned grid, hipStream_t stream) {
  const NormArgs& a = pl.a;
#define RUN(T, VEC, EPT, PLACE, POST, PRE, GATE, MAXT)                       \
  {                                                                          \
    constexpr auto kernel =                                                  \
        &join_bwd_kernel<T, VEC, EPT, PLACE, POST, PRE, GATE, MAXT, false>;  \
    constexpr auto lean =                                                    \
        &join_bwd_kernel<T, VEC, EPT, PLACE, POST, PRE, GATE, MAXT,          \
                         PLACE == kBlock && EPT == 16>;                      \
    const bool is_lean = a.rms && !a.post_bias && !a.pre_bias;               \
    if (grid == 0)                                                           \
      return is_lean ? resident<lean>(pl.threads)                            \
                     : resident<kernel>(pl.threads);                         \
    hipLaunchKernelGGL(is_lean ? lean : kernel, dim3(grid),                  \
                       dim3(pl.threads), 0, stream, a);                      \
    return 1;                                                                \
  }
  BWD_WIDTHS(T, RUN)
#undef RUN
  return 0;
}

#undef BWD_WIDTHS
#undef FWD_WIDTHS
#undef WIDE
#undef NARROW
#undef SIDES
#undef GATES

}  // namespace mamd
