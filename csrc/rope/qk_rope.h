// Host API of the query/key norm and multi-axis rotation kernels (see qk_rope.cu).
#pragma once
#include <ATen/ATen.h>

#include <vector>

namespace h3 {

// q [T, Hq, D], k [T, Hk, D] (bf16 or fp32; k may be absent) -> rotated {q, k}, contiguous.
// With weights ([D], bf16 or fp32) every head is RMS-normalised and scaled first.
// positions [T, A] fp32 and freqs [sum(pairs)] fp32 may be absent (no rotation).
// `status` (int32[4]) takes the reports of the bounds-checked build.
std::vector<at::Tensor> qk_rope_fwd(const at::Tensor& q, const c10::optional<at::Tensor>& k,
                                    const c10::optional<at::Tensor>& q_weight,
                                    const c10::optional<at::Tensor>& k_weight,
                                    const c10::optional<at::Tensor>& positions, const c10::optional<at::Tensor>& freqs,
                                    const std::vector<int64_t>& pairs, bool interleaved, bool inverse, double eps,
                                    const c10::optional<at::Tensor>& status);

// Gradients {dq, dk, dq_weight [D] fp32, dk_weight [D] fp32} of the normalising
// form; dq and dk go into `out` where it has two tensors.
std::vector<at::Tensor> qk_norm_rope_bwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                         const at::Tensor& k_weight, const c10::optional<at::Tensor>& positions,
                                         const c10::optional<at::Tensor>& freqs, const std::vector<int64_t>& pairs,
                                         bool interleaved, const at::Tensor& dq_out, const at::Tensor& dk_out,
                                         double eps, const c10::optional<at::Tensor>& status,
                                         const std::vector<at::Tensor>& out);

}  // namespace h3
