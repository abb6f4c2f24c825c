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
//
// What bounds it: bytes where rows are many - forward 3 tensors, backward 5:
// 1024 x 64 x 1024 bf16 takes 222 us for both, 4.8 TB/s where a copy of 2 GB
// runs at 4.9 (kernels in a profile, where they do not follow each other, 87 +
// 158 at the median), with relu too - and the vector units, at 31 operations
// per element (a third of them the sigmoid), where rows are few: then the time
// axis is split over blocks and a first pass makes the chunks' maps (1 x 16384
// x 1024 bf16: 15 + 21 us forward, 16 + 31 us backward, with relu, whose map
// needs the states, 23 + 31; walked by 4 blocks of 256 channels it took 2700).
// Layout, measured at 1024 x 64 x 1024 backward, each at its best: 32 lanes of
// 2 channels by 2 groups of 8 steps, joined by permlane32_swap, 140 us; 16
// lanes of 4 channels joined by shuffles 176; 64 lanes of 2 channels with 16
// steps 214. Addresses as 64-bit pointers per row, 197 registers for 163, 145.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include <type_traits>

#include "common.h"
#include "fresh.h"
#include "vec.h"

using namespace mamd;

// for lambdas that work on arrays in registers
#define ALWAYS_INLINE __attribute__((always_inline))

namespace {

constexpr int kLC = 32;     // lanes along the channels
constexpr int kSteps = 8;   // steps a thread holds at a time
constexpr int kMaxChunks = 32;

struct ScanArgs {
  const void* x;
  const void* g;
  long xb, xt, gb, gt;      // strides of batch and time, in elements
  const float* state;       // [B,D] or null (zeros)
  const int* lens;          // [B] or null (T)
  float* bnd;               // [B,nt,D] state at each tile's start, or null
  int B, T, D;
  int ctiles;               // channel tiles of a row
  int nt;                   // time tiles
  int nc, tpc;              // chunks of the time axis, tiles in each
  float* agg;               // [2][B,nc,D] the chunks' maps if nc > 1
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

// base (the same in all lanes) + a 32-bit offset per lane, kept in that form:
// left to itself the compiler adds the two and needs a 64-bit address per row
typedef __attribute__((address_space(1))) char gchar;
__device__ __forceinline__ char* uniform(const void* p) {
  const unsigned long v = (unsigned long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return (char*)((unsigned long)hi << 32 | lo);
}
template <typename T, int VEC>
__device__ __forceinline__ vec_t<T, VEC> load_at(const char* base,
                                                 unsigned lane) {
  const gchar* q = (const gchar*)base;
  asm("" : "+s"(q));
  return *(const __attribute__((address_space(1)))
               typename Vec<T, VEC>::mem*)(q + lane);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_at(char* base, unsigned lane,
                                         const float o[VEC]) {
  vec_t<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r[i] = (T)o[i];
  gchar* q = (gchar*)base;
  asm("" : "+s"(q));
  *(__attribute__((address_space(1))) typename Vec<T, VEC>::mem*)(q + lane) =
      r;
}

// Which rows, channels and steps a block works on, and where its lanes are.
// A wave is 32 lanes of VEC channels by 2 groups of kSteps steps; the block's
// NW waves follow each other in time. A lane whose channels would pass the
// row's end moves back to the last VEC channels: it computes what its
// neighbours compute and writes the same values there, so every access is
// whole and in bounds for any D >= VEC.
template <int VEC, int NW>
struct Place {
  static constexpr int kTile = 2 * NW * kSteps;
  int b, chunk, lc, ws, wid, ch, len;
  bool owns;
  size_t vec0;              // this lane in a [B,D] array
  __device__ __forceinline__ Place(const ScanArgs& a, int chunk0) {
    const int lane = threadIdx.x & 63;
    lc = lane & (kLC - 1), ws = lane / kLC;
    wid = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int pair = blockIdx.x % (a.B * a.ctiles);
    chunk = blockIdx.x / (a.B * a.ctiles) + chunk0;
    b = pair / a.ctiles;
    const int c = (pair % a.ctiles) * (kLC * VEC) + lc * VEC;
    owns = c < a.D;
    ch = min(c, a.D - VEC);
    len = __builtin_amdgcn_readfirstlane(
        a.lens ? min(max(a.lens[b], 0), a.T) : a.T);
    vec0 = (size_t)b * a.D + ch;
  }
  // the first of this thread's steps in a tile
  __device__ __forceinline__ int first(int tile) const {
    return tile * kTile + (wid * 2 + ws) * kSteps;
  }
  // Position of step s on the time axis; padded steps (s >= len) come last.
  __device__ __forceinline__ long time_of(const ScanArgs& a, int s) const {
    return a.reverse && s < len ? len - 1 - s : s;
  }
  // A thread's rows of a tile. A wave's rows are read from a scalar base with
  // a 32-bit lane offset (strides are below 2^26 elements), so an address
  // costs no 64-bit arithmetic per lane and no register per row.
  // FULL: every step exists; otherwise rows behind the sequence repeat its
  // last one.
  template <bool FULL, typename T>
  __device__ __forceinline__ void load(const ScanArgs& a, const T* base,
                                       long stride, int tile,
                                       vec_t<T, VEC> r[kSteps]) const {
    const int sw = tile * kTile + wid * 2 * kSteps;
    const long bytes = stride * (long)sizeof(T);
    if constexpr (FULL) {
      const long d = a.reverse ? -bytes : bytes;
      const int t0 = a.reverse ? len - 1 - kSteps - sw : sw;
      const char* q = uniform((const char*)base + t0 * bytes);
      const unsigned lane = (unsigned)((a.reverse ? 1 - ws : ws) * kSteps) *
                                (unsigned)bytes +
                            (unsigned)ch * (unsigned)sizeof(T);
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        r[j] = load_at<T, VEC>(q + j * d, lane);
    } else {
      const int t0 = a.reverse ? max(len - sw - 2 * kSteps, 0)
                               : min(sw, len - 1);
      const char* q = uniform((const char*)base + t0 * bytes);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int t = time_of(a, min(sw + ws * kSteps + j, len - 1));
        const unsigned lane = (unsigned)(t - t0) * (unsigned)bytes +
                              (unsigned)ch * (unsigned)sizeof(T);
        r[j] = load_at<T, VEC>(q, lane);
      }
    }
  }
  // FULL == false: up to T, padding included
  template <bool FULL, typename T>
  __device__ __forceinline__ void store(const ScanArgs& a, T* base,
                                        long stride, int tile,
                                        const float o[kSteps][VEC]) const {
    const int sw = tile * kTile + wid * 2 * kSteps;
    const long bytes = stride * (long)sizeof(T);
    if constexpr (FULL) {
      const long d = a.reverse ? -bytes : bytes;
      const int t0 = a.reverse ? len - 1 - kSteps - sw : sw;
      char* q = uniform((char*)base + t0 * bytes);
      const unsigned lane = (unsigned)((a.reverse ? 1 - ws : ws) * kSteps) *
                                (unsigned)bytes +
                            (unsigned)ch * (unsigned)sizeof(T);
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        store_at<T, VEC>(q + j * d, lane, o[j]);
    } else {
      const int s0 = sw + ws * kSteps;
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
        if (s0 + j < a.T)
          store_vec<T, VEC>(base + time_of(a, s0 + j) * stride + ch, o[j]);
    }
  }
};

// the value of the wave's lower and of its upper half, in all lanes
__device__ __forceinline__ void halves(float v, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v),
                                                  __float_as_uint(v), false,
                                                  false);
  lo = __uint_as_float(r[0]);
  hi = __uint_as_float(r[1]);
}

// From a group's map (A, H): the wave's map, and in eA, eH the map of the
// steps of its wave that come before this group's.
template <int VEC>
__device__ __forceinline__ void wave_fold(int ws, float A[VEC], float H[VEC],
                                          float eA[VEC], float eH[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float a0, a1, h0, h1;
    halves(A[v], a0, a1);
    halves(H[v], h0, h1);
    A[v] = a1 * a0;
    H[v] = a1 * h0 + h1;
    eA[v] = ws ? a0 : 1.f;
    eH[v] = ws ? h0 : 0.f;
  }
}

// the same from the far end
template <int VEC>
__device__ __forceinline__ void wave_fold_back(int ws, float A[VEC],
                                               float M[VEC], float eA[VEC],
                                               float eM[VEC]) {
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    float a0, a1, m0, m1;
    halves(A[v], a0, a1);
    halves(M[v], m0, m1);
    A[v] = a0 * a1;
    M[v] = a0 * m1 + m0;
    eA[v] = ws ? 1.f : a1;
    eM[v] = ws ? 0.f : m1;
  }
}

// a NaN state stays visible, which fmaxf would turn into 0
__device__ __forceinline__ float activate(float c, int relu) {
  return relu && c < 0.f ? 0.f : c;
}

// calls fn with a compile-time truth value
template <typename F>
__device__ __forceinline__ void with_bool(bool v, F fn) {
  if (v) fn(std::true_type{});
  else fn(std::false_type{});
}

// The maps of the chunks [k0, k1) from the aggregates, applied to c: every
// wave folds some of them, one channel per lane, and the waves' maps meet in
// LDS. back: from the last chunk to the first.
template <int VEC, int NW>
__device__ __forceinline__ void fold_chunks(const ScanArgs& a,
                                            const Place<VEC, NW>& p, int k0,
                                            int k1, bool back,
                                            float (*sA)[kLC * VEC],
                                            float (*sH)[kLC * VEC],
                                            float c[VEC]) {
  constexpr int PER = (kMaxChunks + NW - 1) / NW;
  const int lane = threadIdx.x & 63, n = k1 - k0;
  if (lane < kLC * VEC) {
    const int c0 = p.b * a.ctiles;  // this block's pair, without its channels
    const int pair = blockIdx.x % (a.B * a.ctiles) - c0;
    const int ch = min(min(pair * (kLC * VEC) + (lane / VEC) * VEC,
                           a.D - VEC) + lane % VEC, a.D - 1);
    const size_t plane = (size_t)a.B * a.nc * a.D;
    float va[PER], vh[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {  // r-th map to apply; past n: the last
      const int r = min(p.wid * PER + i, n - 1);
      const float* q =
          a.agg + ((size_t)p.b * a.nc + (back ? k1 - 1 - r : k0 + r)) * a.D +
          ch;
      va[i] = q[0];
      vh[i] = q[plane];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (p.wid * PER + i >= n) va[i] = 1.f, vh[i] = 0.f;
    float A = 1.f, H = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) H = va[i] * H + vh[i], A *= va[i];
    sA[p.wid][lane] = A;
    sH[p.wid][lane] = H;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int v = 0; v < VEC; ++v)
      c[v] = sA[w][p.lc * VEC + v] * c[v] + sH[w][p.lc * VEC + v];
  __syncthreads();
}

// AGG: only the chunk's map, for the blocks of the pass that follows.
template <typename T, int VEC, int NW, bool AGG>
__global__ __launch_bounds__(NW * 64) void scan_fwd_kernel(ScanArgs a) {
  __shared__ float sA[2][NW][kLC * VEC], sH[2][NW][kLC * VEC];
  using P = Place<VEC, NW>;
  const P p(a, 0);
  const T* x = (const T*)a.x + (size_t)p.b * a.xb;
  const T* g = (const T*)a.g + (size_t)p.b * a.gb;
  T* y = (T*)a.y + (size_t)p.b * a.T * a.D;
  const int k0 = p.chunk * a.tpc, k1 = min(k0 + a.tpc, a.nt);
  // tiles full of steps, and tiles with a step; what follows is padding
  const int kf = min(k1, p.len / P::kTile);
  const int kv = min(k1, (p.len + P::kTile - 1) / P::kTile);

  vec_t<T, VEC> xr[kSteps], gr[kSteps];
  auto fetch = [&](int tile, auto full) ALWAYS_INLINE {
    constexpr bool FULL = decltype(full)::value;
    p.template load<FULL>(a, x, a.xt, tile, xr);
    p.template load<FULL>(a, g, a.gt, tile, gr);
  };
  if (k0 < kf) fetch(k0, std::true_type{});

  float c[VEC], Ap[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    c[v] = !AGG && a.state ? a.state[p.vec0 + v] : 0.f;
    Ap[v] = 1.f;
  }
  if (!AGG && p.chunk > 0)
    fold_chunks<VEC, NW>(a, p, 0, p.chunk, false, sA[0], sH[0], c);

  auto body = [&](int tile, auto full) ALWAYS_INLINE {
    constexpr bool FULL = decltype(full)::value;
    const int s0 = p.first(tile), buf = tile & 1;
    if (!AGG && a.bnd && threadIdx.x < kLC && p.owns)
      store_vec<float, VEC>(a.bnd + ((size_t)p.b * a.nt + tile) * a.D + p.ch,
                            c);
    float f[kSteps][VEC], h[kSteps][VEC];
    float A[VEC], H[VEC], eA[VEC], eH[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const bool on = FULL || s0 + j < p.len;
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
    if (FULL && tile + 1 < kf) fetch(tile + 1, full);
    wave_fold<VEC>(p.ws, A, H, eA, eH);
    if (p.ws == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        sA[buf][p.wid][p.lc * VEC + v] = A[v];
        sH[buf][p.wid][p.lc * VEC + v] = H[v];
      }
    }
    __syncthreads();
    float cur[VEC];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (w == p.wid) cur[v] = c[v];
        const float wa = sA[buf][w][p.lc * VEC + v];
        c[v] = wa * c[v] + sH[buf][w][p.lc * VEC + v];
        if constexpr (AGG) Ap[v] *= wa;
      }
    if constexpr (!AGG) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) cur[v] = eA[v] * cur[v] + eH[v];
      with_bool(a.relu, [&](auto relu) ALWAYS_INLINE {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            cur[v] = f[j][v] * cur[v] + h[j][v];
            h[j][v] = activate(cur[v], decltype(relu)::value);
          }
      });
      if constexpr (!FULL) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            if (s0 + j >= p.len) h[j][v] = 0.f;
      }
      if (p.owns) p.template store<FULL>(a, y, (long)a.D, tile, h);
    }
  };
  for (int tile = k0; tile < kf; ++tile) body(tile, std::true_type{});
  if (k0 < kv && kf < kv) {
    fetch(kv - 1, std::false_type{});
    body(kv - 1, std::false_type{});
  }
  if constexpr (AGG) {
    if (threadIdx.x < kLC && p.owns) {
      float* q = a.agg + ((size_t)p.b * a.nc + p.chunk) * a.D + p.ch;
      store_vec<float, VEC>(q, Ap);
      store_vec<float, VEC>(q + (size_t)a.B * a.nc * a.D, c);
    }
  } else {
    const float zero[VEC] = {};
    for (int tile = max(kv, k0); tile < k1; ++tile) {
      if (a.bnd && threadIdx.x < kLC && p.owns)
        store_vec<float, VEC>(
            a.bnd + ((size_t)p.b * a.nt + tile) * a.D + p.ch, c);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int s = p.first(tile) + j;
        if (s < a.T && p.owns) store_vec<T, VEC>(y + (size_t)s * a.D + p.ch, zero);
      }
    }
    if (p.chunk == a.nc - 1 && threadIdx.x < kLC && p.owns)
      store_vec<float, VEC>(a.last + p.vec0, c);
  }
}

// AGG: only the chunk's map of mu.
template <typename T, int VEC, int NW, bool AGG>
__global__ __launch_bounds__(NW * 64) void scan_bwd_kernel(ScanArgs a) {
  __shared__ float sA[2][NW][kLC * VEC], sH[2][NW][kLC * VEC];
  __shared__ float sM[2][NW][kLC * VEC];
  using P = Place<VEC, NW>;
  const P p(a, AGG ? 1 : 0);
  const T* x = (const T*)a.x + (size_t)p.b * a.xb;
  const T* g = (const T*)a.g + (size_t)p.b * a.gb;
  const T* dy =
      a.dy ? (const T*)a.dy + (size_t)p.b * a.T * a.D : nullptr;
  T* dx = (T*)a.dx + (size_t)p.b * a.dxb;
  T* dg = (T*)a.dg + (size_t)p.b * a.dgb;
  const int k0 = p.chunk * a.tpc, k1 = min(k0 + a.tpc, a.nt);
  const int kf = min(k1, p.len / P::kTile);
  const int kv = min(k1, (p.len + P::kTile - 1) / P::kTile);
  // the map of mu needs the states for relu's side only
  const bool states = !AGG || a.relu;

  vec_t<T, VEC> xr[kSteps], gr[kSteps], dr[kSteps];
  float cr[VEC];            // the state at the tile's start
#pragma unroll
  for (int j = 0; j < kSteps; ++j) xr[j] = dr[j] = {};
  auto fetch = [&](int tile, auto full) ALWAYS_INLINE {
    constexpr bool FULL = decltype(full)::value;
    if (states) p.template load<FULL>(a, x, a.xt, tile, xr);
    p.template load<FULL>(a, g, a.gt, tile, gr);
    if (dy) p.template load<FULL>(a, dy, (long)a.D, tile, dr);
    const float* cp =
        a.bnd ? a.bnd + ((size_t)p.b * a.nt + tile) * a.D + p.ch
              : (a.state ? a.state + p.vec0 : nullptr);
#pragma unroll
    for (int v = 0; v < VEC; ++v) cr[v] = cp && states ? cp[v] : 0.f;
  };
  const bool rest = k0 < kv && kf < kv;  // the last of them is not full
  if (rest)
    fetch(kv - 1, std::false_type{});
  else if (k0 < kf)
    fetch(kf - 1, std::true_type{});

  float mu[VEC], Ap[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    mu[v] = !AGG && a.dlast ? a.dlast[p.vec0 + v] : 0.f;
    Ap[v] = 1.f;
  }
  if (!AGG && p.chunk < a.nc - 1)
    fold_chunks<VEC, NW>(a, p, p.chunk + 1, a.nc, true, sA[0], sH[0], mu);

  if constexpr (!AGG) {
    const float zero[VEC] = {};
    for (int tile = max(kv, k0); tile < k1; ++tile)
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int s = p.first(tile) + j;
        if (s < a.T && p.owns) {
          store_vec<T, VEC>(dx + (size_t)s * a.dxt + p.ch, zero);
          store_vec<T, VEC>(dg + (size_t)s * a.dgt + p.ch, zero);
        }
      }
  }
  auto body = [&](int tile, auto full) ALWAYS_INLINE {
    constexpr bool FULL = decltype(full)::value;
    const int s0 = p.first(tile), buf = tile & 1;
    float f[kSteps][VEC], om[kSteps][VEC], w[kSteps][VEC], d[kSteps][VEC];
    float A[VEC], H[VEC], A2[VEC], eA[VEC], eH[VEC], c[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) A[v] = 1.f, H[v] = 0.f, c[v] = cr[v];
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      const bool on = FULL || s0 + j < p.len;
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
    if (tile > k0) fetch(tile - 1, std::true_type{});
#pragma unroll
    for (int v = 0; v < VEC; ++v) A2[v] = A[v];
    if (states) {
      wave_fold<VEC>(p.ws, A, H, eA, eH);
      if (p.ws == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          sA[buf][p.wid][p.lc * VEC + v] = A[v];
          sH[buf][p.wid][p.lc * VEC + v] = H[v];
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NW - 1; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v)
          if (k < p.wid)
            c[v] = sA[buf][k][p.lc * VEC + v] * c[v] +
                   sH[buf][k][p.lc * VEC + v];
#pragma unroll
      for (int v = 0; v < VEC; ++v) c[v] = eA[v] * c[v] + eH[v];
      // w becomes c_{t-1} - x_t, d is cut where relu was off
      with_bool(a.relu, [&](auto relu) ALWAYS_INLINE {
#pragma unroll
        for (int j = 0; j < kSteps; ++j)
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            const float xv = w[j][v];
            w[j][v] = c[v] - xv;
            c[v] = f[j][v] * c[v] + om[j][v] * xv;
            if (decltype(relu)::value && c[v] <= 0.f) d[j][v] = 0.f;
          }
      });
    }
    // this thread's steps from the far end, with nothing coming in
    float M[VEC], eM[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) M[v] = 0.f;
#pragma unroll
    for (int j = kSteps - 1; j >= 0; --j)
#pragma unroll
      for (int v = 0; v < VEC; ++v) M[v] = f[j][v] * (d[j][v] + M[v]);
    wave_fold_back<VEC>(p.ws, A2, M, eA, eM);
    if (p.ws == 0) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        sM[buf][p.wid][p.lc * VEC + v] = M[v];
        if (!states) sA[buf][p.wid][p.lc * VEC + v] = A2[v];
      }
    }
    __syncthreads();
    float cur[VEC];
#pragma unroll
    for (int k = NW - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        if (k == p.wid) cur[v] = mu[v];
        const float wa = sA[buf][k][p.lc * VEC + v];
        mu[v] = wa * mu[v] + sM[buf][k][p.lc * VEC + v];
        if constexpr (AGG) Ap[v] *= wa;
      }
    if constexpr (!AGG) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) cur[v] = eA[v] * cur[v] + eM[v];
#pragma unroll
      for (int j = kSteps - 1; j >= 0; --j) {
        const bool on = FULL || s0 + j < p.len;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float lam = d[j][v] + cur[v];
          cur[v] = f[j][v] * lam;
          d[j][v] = on ? om[j][v] * lam : 0.f;
          w[j][v] = on ? cur[v] * om[j][v] * w[j][v] : 0.f;
        }
      }
      if (p.owns) {
        p.template store<FULL>(a, dx, a.dxt, tile, d);
        p.template store<FULL>(a, dg, a.dgt, tile, w);
      }
    }
  };
  if (rest) body(kv - 1, std::false_type{});
  for (int tile = kf - 1; tile >= k0; --tile) body(tile, std::true_type{});
  if constexpr (AGG) {
    if (threadIdx.x < kLC && p.owns) {
      float* q = a.agg + ((size_t)p.b * a.nc + p.chunk) * a.D + p.ch;
      store_vec<float, VEC>(q, Ap);
      store_vec<float, VEC>(q + (size_t)a.B * a.nc * a.D, mu);
    }
  } else if (a.dstate && p.chunk == 0 && threadIdx.x < kLC && p.owns) {
    store_vec<float, VEC>(a.dstate + p.vec0, mu);
  }
}

// One token for each row: the recurrence at T = 1, on a pool of states. Bound
// by bytes (4096 x 1024 bf16: 10.6 us, 5.6 TB/s) or by the launch (4 rows: 2).
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

// 16 steps a wave: 4 waves make the tile of 64, one is enough for 16 steps
int waves_of(int T) { return T <= 16 ? 1 : 4; }
int vec_of_width(int D) { return D >= 2 ? 2 : 1; }

// the kernels' lane offsets are 32 bits over 16 rows
long time_stride(const torch::Tensor& t) {
  if (t.size(1) <= 1) return 0;
  TORCH_CHECK(t.stride(1) < (1L << 26),
              "gated_scan: time strides must stay below 2^26 elements");
  return t.stride(1);
}

ScanArgs base_args(const torch::Tensor& x, const torch::Tensor& g,
                   const c10::optional<torch::Tensor>& state,
                   const c10::optional<torch::Tensor>& lens, bool reverse,
                   bool relu) {
  check_rows(x, g, "gated_scan");
  TORCH_CHECK(x.dim() == 3, "gated_scan: x must be [B, T, D]");
  TORCH_CHECK(x.size(0) < (1 << 30) && x.size(1) < (1 << 30) &&
                  x.size(2) < (1 << 26),
              "gated_scan: B and T must stay below 2^30, D below 2^26");
  ScanArgs a{};
  a.x = x.data_ptr();
  a.g = g.data_ptr();
  a.xb = x.stride(0), a.xt = time_stride(x);
  a.gb = g.stride(0), a.gt = time_stride(g);
  a.state = state_ptr(state, x, "state");
  a.lens = lens_ptr(lens, x);
  a.B = x.size(0), a.T = x.size(1), a.D = x.size(2);
  // a tile holds 16 steps per wave; short sequences take fewer waves. The
  // forward and the backward pass get the same tiles, since one keeps the
  // states that the other starts from.
  const int tile = 2 * kSteps * waves_of(a.T);
  a.ctiles = (a.D + vec_of_width(a.D) * kLC - 1) / (vec_of_width(a.D) * kLC);
  a.nt = (a.T + tile - 1) / tile;
  const long pairs = (long)a.B * a.ctiles;
  // The chunks' maps cost another reading of the inputs, so the time axis is
  // split only where blocks that walk all of it are few. Forward and backward
  // with relu at 2048 x 1024, split and walked: bf16 8 sequences (128 blocks)
  // 90 and 125 us, 10 104 and 125, 12 131 and 126, 16 159 and 130; fp32 8 159
  // and 167, 10 189 and 176, 12 235 and 185; 12 x 16384 x 1024 bf16 1139 and
  // 945. Up to two blocks per CU, in at most 32 chunks: fewer than 16 tiles of
  // channels leave CUs without one (1 x 16384 x 64: 64 us, walked 896).
  const int nc = pairs >= 192 || pairs == 0
                     ? 1
                     : (int)std::min<long>({kMaxChunks, (long)a.nt,
                                            (512 + pairs - 1) / pairs});
  a.tpc = nc > 1 ? (a.nt + nc - 1) / nc : std::max(a.nt, 1);
  a.nc = std::max((a.nt + a.tpc - 1) / a.tpc, 1);
  TORCH_CHECK(pairs < (1L << 31), "gated_scan: too many rows");
  a.reverse = reverse;
  a.relu = relu;
  return a;
}

#define SCAN_DTYPES(st, FN)                                         \
  if (st == torch::kBFloat16) { FN(bf16_t); }                       \
  else if (st == torch::kHalf) { FN(f16_t); }                       \
  else if (st == torch::kFloat32) { FN(float); }                    \
  else TORCH_CHECK(false, "gated_scan: unsupported dtype");

template <bool AGG>
void launch(bool bwd, const torch::Tensor& x, const ScanArgs& a,
            hipStream_t stream) {
  // no chunk follows the last one (backward: the first): its map is not used
  const long blocks = (long)a.B * a.ctiles * (AGG ? a.nc - 1 : a.nc);
  const int nw = waves_of(a.T);
  TORCH_CHECK(blocks * nw * 64 < (1L << 32), "gated_scan: too many rows");
  const dim3 grid((unsigned)blocks);
#define RUN2(ET, VEC, NW)                                                    \
  if (bwd)                                                                   \
    hipLaunchKernelGGL((scan_bwd_kernel<ET, VEC, NW, AGG>), grid,            \
                       dim3(NW * 64), 0, stream, a);                         \
  else                                                                       \
    hipLaunchKernelGGL((scan_fwd_kernel<ET, VEC, NW, AGG>), grid,            \
                       dim3(NW * 64), 0, stream, a)
// one wave holds all of the steps: there are no chunks
#define RUN1(ET, VEC)                                                        \
  if (nw == 1) {                                                             \
    TORCH_CHECK(!AGG, "gated_scan: no such chunks");                         \
    if constexpr (!AGG) { RUN2(ET, VEC, 1); }                                \
  } else { RUN2(ET, VEC, 4); }
#define RUN(ET)                                                              \
  if (vec_of_width(a.D) == 2) { RUN1(ET, 2) } else { RUN1(ET, 1) }
  SCAN_DTYPES(x.scalar_type(), RUN)
#undef RUN
#undef RUN1
#undef RUN2
  C10_HIP_KERNEL_LAUNCH_CHECK();
}

void run(bool bwd, const torch::Tensor& x, ScanArgs& a) {
  auto stream = at::cuda::getCurrentHIPStream();
  torch::Tensor agg;
  if (a.nc > 1) {
    agg = fresh({2, a.B, a.nc, a.D}, torch::kFloat32, x);
    a.agg = agg.data_ptr<float>();
    launch<true>(bwd, x, a, stream);
  }
  launch<false>(bwd, x, a, stream);
}

}  // namespace

// returns (y, last, bnd); bnd is undefined unless want_bnd and T spans tiles
std::vector<torch::Tensor> gated_scan_fwd(torch::Tensor x, torch::Tensor gate,
                                          c10::optional<torch::Tensor> state,
                                          c10::optional<torch::Tensor> lens,
                                          bool reverse, bool relu,
                                          bool want_bnd) {
  ScanArgs a = base_args(x, gate, state, lens, reverse, relu);
  const c10::DeviceGuard guard(x.device());
  auto y = fresh_like(x);
  auto last = fresh({a.B, a.D}, torch::kFloat32, x);
  torch::Tensor bnd;
  if (want_bnd && a.nt > 1) {
    bnd = fresh({a.B, a.nt, a.D}, torch::kFloat32, x);
    a.bnd = bnd.data_ptr<float>();
  }
  a.y = y.data_ptr();
  a.last = last.data_ptr<float>();
  if (a.B == 0) return {y, last, bnd};
  run(false, x, a);
  return {y, last, bnd};
}

// writes dx and dgate (any batch and time strides); returns dstate, undefined
// unless want_dstate
torch::Tensor gated_scan_bwd(torch::Tensor x, torch::Tensor gate,
                             c10::optional<torch::Tensor> state,
                             c10::optional<torch::Tensor> lens,
                             torch::Tensor bnd,
                             c10::optional<torch::Tensor> dy,
                             c10::optional<torch::Tensor> dlast, bool reverse,
                             bool relu, torch::Tensor dx,
                             torch::Tensor dgate, bool want_dstate) {
  ScanArgs a = base_args(x, gate, state, lens, reverse, relu);
  const c10::DeviceGuard guard(x.device());
  check_rows(dx, dgate, "gated_scan_bwd");
  TORCH_CHECK(dx.sizes() == x.sizes() && dx.device() == x.device() &&
                  dx.scalar_type() == x.scalar_type(),
              "gated_scan_bwd: dx must be like x");
  if (a.nt > 1) {
    TORCH_CHECK(bnd.defined() && bnd.device() == x.device() &&
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
  a.dxb = dx.stride(0), a.dxt = time_stride(dx);
  a.dgb = dgate.stride(0), a.dgt = time_stride(dgate);
  torch::Tensor dstate;
  if (want_dstate) {
    dstate = fresh({a.B, a.D}, torch::kFloat32, x);
    a.dstate = dstate.data_ptr<float>();
  }
  if (a.B == 0) return dstate;
  run(true, x, a);
  return dstate;
}

// one step for N rows; state_out may be state itself
torch::Tensor gated_step_fwd(torch::Tensor x, torch::Tensor gate,
                             torch::Tensor state, torch::Tensor state_out,
                             bool relu) {
  check_rows(x, gate, "gated_step");
  TORCH_CHECK(x.dim() == 2, "gated_step: x must be [N, D]");
  const float* sp = state_ptr(state, x, "state");
  state_ptr(state_out, x, "state_out");
  const c10::DeviceGuard guard(x.device());
  const long N = x.size(0), D = x.size(1);
  TORCH_CHECK(D < (1L << 30), "gated_step: the width must stay below 2^30");
  auto y = fresh_like(x);
  if (N == 0) return y;
  auto stream = at::cuda::getCurrentHIPStream();
  const int vpr = (int)((D + 3) / 4);
  const long n_vec = N * vpr;
  const long grid = (n_vec + 255) / 256;
  TORCH_CHECK(grid * 256 < (1L << 32), "gated_step: too many rows");
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
