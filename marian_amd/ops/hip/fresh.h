// Uninitialised device tensors without the dispatcher (about 0.5 us each
// where torch::empty takes 1.4): small calls are bound by the host.
#pragma once

#include <ATen/hip/EmptyTensor.h>

namespace mamd {

inline at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype,
                        const at::Tensor& beside) {
  return at::detail::empty_cuda(sizes, dtype, beside.device(), std::nullopt);
}
inline at::Tensor fresh_like(const at::Tensor& t) {
  return fresh(t.sizes(), t.scalar_type(), t);
}

}  // namespace mamd
