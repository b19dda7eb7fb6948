// Host helpers for tensors [tokens, heads, head_dim] whose rows kernels read as they lie.
#pragma once
#include <ATen/ATen.h>

#include <cstdint>

namespace h3 {

// `t` itself if the kernels can read its layout (unit stride within a head,
// every head on a 16-byte boundary, no zero stride), else a copy, which starts on such a boundary.
// Not contiguous(): a contiguous tensor off the boundary would come back as it is.
inline at::Tensor fit(const at::Tensor& t) {
  if (!t.is_cuda() || t.dim() != 3 || t.numel() == 0) return t;
  const int64_t unit = 16 / t.element_size();
  const bool fits = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 &&
                    (t.size(0) == 1 || (t.stride(0) > 0 && t.stride(0) % unit == 0)) &&
                    (t.size(1) == 1 || (t.stride(1) > 0 && t.stride(1) % unit == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

}  // namespace h3
