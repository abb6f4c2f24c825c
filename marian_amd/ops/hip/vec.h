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
// 16-bit inputs take the hardware's exp2 and reciprocal (about 1 ulp of 32
// bits each, 2^-14 of a bf16 step); 32-bit inputs take the library's.
template <typename T>
__device__ __forceinline__ void sigmoid2(float g, float& f, float& om) {
  float e, r;
  if constexpr (sizeof(T) == 4) {
    e = expf(-fabsf(g));
    r = 1.f / (1.f + e);
  } else {
    e = __builtin_amdgcn_exp2f(-1.4426950408889634f * fabsf(g));
    r = __builtin_amdgcn_rcpf(1.f + e);
  }
  const float s = e * r;
  f = g >= 0.f ? r : s;
  om = g >= 0.f ? s : r;
}

}  // namespace mamd
