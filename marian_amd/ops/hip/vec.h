// Vectors of VEC elements at any element alignment.
// gfx950 global loads and stores take addresses that are aligned to the
// element only, so rows of an odd width keep the wide access: a type that
// promises no more than that still compiles to one dwordx2 / dwordx4.
#pragma once

#include <hip/hip_runtime.h>

namespace mamd {

using bf16_t = __bf16;
using f16_t = _Float16;

template <typename T, int VEC>
struct Vec {
  typedef T type __attribute__((ext_vector_type(VEC)));
  typedef T mem __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
};
template <typename T, int VEC>
using vec_t = typename Vec<T, VEC>::type;

template <typename T, int VEC>
__device__ __forceinline__ vec_t<T, VEC> load_vec(const T* p) {
  return *reinterpret_cast<const typename Vec<T, VEC>::mem*>(p);
}

// one rounding to nearest even per element
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float o[VEC]) {
  vec_t<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r[i] = (T)o[i];
  *reinterpret_cast<typename Vec<T, VEC>::mem*>(p) = r;
}

// f = sigmoid(g) and om = 1 - f, each to its own relative precision: with
// e = exp(-|g|) they are 1/(1+e) and e/(1+e), neither of which cancels.
// e is the hardware's exp2 of t = -|g| log2(e). 16-bit inputs take it and the
// hardware's reciprocal as they are: t's rounding is worth |g| units of 32
// bits, 2^-12 of a bf16 step at |g| = 16, and new states are as near to 64 bits
// as with the longer form (3.3e-8 - 5.8e-8 of them, |g| from 0.5 to 16), which
// costs a bound scan 10 - 12 %. 32-bit inputs add what t's rounding
// left out, and one Newton step to the reciprocal: about 2 units, in half the
// instructions of a library exp and divide (1.4 times the scan's speed).
template <typename T>
__device__ __forceinline__ void sigmoid2(float g, float& f, float& om) {
  constexpr float kL2 = 1.44269504f, kL2Lo = 1.92596299e-8f;  // log2(e)
  float a = fabsf(g), e, r;
  if constexpr (sizeof(T) == 4) {
    a = a > 200.f ? 200.f : a;  // e is 0 from there on; NaN stays
    const float t = a * kL2;
    const float lo = fmaf(a, kL2Lo, fmaf(a, kL2, -t));
    e = __builtin_amdgcn_exp2f(-t);
    e = fmaf(e * lo, -0.693147181f, e);
    const float d = 1.f + e;
    r = __builtin_amdgcn_rcpf(d);
    r = fmaf(fmaf(-d, r, 1.f), r, r);
  } else {
    e = __builtin_amdgcn_exp2f(-kL2 * a);
    r = __builtin_amdgcn_rcpf(1.f + e);
  }
  const float s = e * r;
  f = g >= 0.f ? r : s;
  om = g >= 0.f ? s : r;
}

}  // namespace mamd
