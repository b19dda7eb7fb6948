// Host API of attention over packed sequences (see packed.h for the layout).
#pragma once
#include <ATen/ATen.h>

#include <tuple>
#include <vector>

namespace h3 {

// Work lists of a packed batch for a GPU with `sms` multiprocessors, on the CPU:
// {int32 blob, meta}.  The blob goes to the device once; both are passed to every call.
std::tuple<at::Tensor, std::vector<int64_t>> packed_schedule(const std::vector<int64_t>& q_lens,
                                                             const std::vector<int64_t>& k_lens, int64_t heads,
                                                             int64_t kv_heads, int64_t head_dim, bool causal,
                                                             int64_t sms);

// q [Tq, Hq, D], k, v [Tk, Hk, D] bf16 -> {o [Tq, Hq, D] bf16, lse [Hq, Tq] fp32 (natural log)}
std::vector<at::Tensor> attention_packed_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             const at::Tensor& blob, const std::vector<int64_t>& meta, double scale,
                                             const at::Tensor& status, int64_t limit_ns);

// Gradients {dq, dk, dv}, written into `out` where it has three tensors.
std::vector<at::Tensor> attention_packed_bwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             const at::Tensor& o, const at::Tensor& lse, const at::Tensor& dout,
                                             const at::Tensor& blob, const std::vector<int64_t>& meta, double scale,
                                             const at::Tensor& status, int64_t limit_ns,
                                             const std::vector<at::Tensor>& out);

}  // namespace h3
